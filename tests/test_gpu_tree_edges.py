"""eid_attn_tree where a rule or a number reaches its end, with lse and without (two kernels: exact
fp32 row sums, and row sums of the rounded weights from the matrix unit).

Tolerance, with A = sum w |v| / sum w >= |out| beside the reference: the numerator's weights are rounded to
bf16 (2^-8 A), without lse the denominator's as well (2^-8 |out|), the output once more (2^-8 |out|);
fp32 sums, exponentials and the fp16 pieces of a cut context stay below 2^-8 A / 2.  So |error| <= 2.5 * 2^-8 A
with lse, 3.5 * 2^-8 A without.  lse: |error| <= 1e-5 (1 + |lse|)."""
import numpy as np
import pytest
import torch

import eidola_amd as ea
from eidola_amd import KV_BF16, KV_FP8_E4M3, synth

import cache_ref as R
from helpers import cpu_caches, fp8_scales, logical_tensors, make_batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def G():
    import gpu_helpers
    assert torch.cuda.is_available()
    ea.load_library()
    return gpu_helpers


def reference(b, q, kc, vc, mask, sinks, ks=None, vs=None):
    """(out, lse, A) in 64 bits, a KV head's rows at once."""
    outs, lses, mags = [], [], []
    for s in range(b.num_seqs):
        x, y = b.cu_seqlens_q[s], b.cu_seqlens_q[s + 1]
        n = int(y - x)
        see = R.tree_visible(mask[x:y], n, int(b.seq_lens[s]), b.geom.window)
        k, v = R.cache_rows(b, kc, ks, s), R.cache_rows(b, vc, vs, s)
        out, mag = np.zeros((2, n, b.geom.num_q_heads, 64))
        lse = np.full((n, b.geom.num_q_heads), -np.inf)
        for h in range(b.geom.num_q_heads):
            sc = np.where(see, R.f64(q[x:y, h]) @ k[:, h // 8].T * b.geom.softmax_scale, -np.inf)
            sink = -np.inf if sinks is None else float(sinks[h])
            top = np.maximum(sc.max(1), sink)
            some = top > -np.inf
            p = np.exp(sc[some] - top[some, None])
            den = p.sum(1) + np.exp(sink - top[some])
            out[some, h] = p @ v[:, h // 8] / den[:, None]
            mag[some, h] = p @ np.abs(v[:, h // 8]) / den[:, None]
            lse[some, h] = top[some] + np.log(den)
        outs.append(out)
        lses.append(lse)
        mags.append(mag)
    return np.concatenate(outs), np.concatenate(lses), np.concatenate(mags)


def check(G, b, q, kc, vc, mask, sinks, ks=None, vs=None):
    ref, ref_lse, mag = reference(b, q, kc, vc, mask, sinks, ks, vs)
    for with_lse in (True, False):
        out = ea.attn_tree(b.geom, G.bf16_dev(q), G.cache_dev(kc), G.cache_dev(vc), G.dev(b.block_table),
                           G.dev(b.seq_lens), G.dev(b.cu_seqlens_q), G.dev(mask), max_q_len=b.max_q_len,
                           max_kv_len=b.max_kv_len, sinks=G.dev(sinks), k_scale=G.dev(ks), v_scale=G.dev(vs),
                           return_lse=with_lse)
        if with_lse:
            l = out[1].cpu().numpy().astype(np.float64)
            assert np.array_equal(np.isinf(l), np.isinf(ref_lse))
            fine = np.isfinite(ref_lse)
            assert (np.abs(l[fine] - ref_lse[fine]) <= 1e-5 * (1 + np.abs(ref_lse[fine]))).all()
            out = out[0]
        got = R.f64(G.bits_host(out))
        tol = (2.5 if with_lse else 3.5) * R.BF16_HALF_STEP * mag + 1e-6
        assert np.isfinite(got).all() and (np.abs(got - ref) <= tol).all(), float((np.abs(got - ref) / tol).max())


@pytest.mark.parametrize("kv_dtype", [KV_BF16, KV_FP8_E4M3])
@pytest.mark.parametrize("n", [1, 2, 12, 17, 32, 33, 70])
def test_a_window_as_long_as_the_tree(G, n, kv_dtype):
    # A token with an empty mask stands at depth -1, n positions before a row that sees all n tokens: a window of
    # n hides it from that row, one of n + 1 does not.
    for window in (n - 1, n, n + 1):
        if window == 0:
            continue
        b, q, kc, vc, ks, vs, sinks = R.filled([n + 150, n], [n, n], window=window, kv_dtype=kv_dtype, num_kv_heads=2)
        rng = np.random.default_rng(n)
        ints = [int.from_bytes(rng.bytes(9), "little") & ((1 << n) - 1) for _ in range(2 * n)]
        for first in (0, n):
            ints[first] = ints[first + n // 2] = 0
            ints[first + n - 1] = (1 << n) - 1
        check(G, b, q, kc, vc, R.masks_from_ints(ints, (n + 63) // 64), sinks, ks, vs)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 150])
@pytest.mark.parametrize("n", [100, 200])
def test_windows_that_nothing_outgrows(G, n, window):
    # the largest windows that a descriptor holds, drafted tokens more than a chunk behind a short context
    b, q, kc, vc, ks, vs, sinks = R.filled([n + 10, n], [n, n], window=window, num_kv_heads=1)
    rng = np.random.default_rng(n)
    check(G, b, q, kc, vc, R.tree_masks([R.random_parents(n, rng), list(range(-1, n - 1))], (n + 63) // 64), sinks)


@pytest.mark.parametrize("n", [4, 12, 20, 30])
def test_small_values_behind_a_cut_context_leave_its_sums_alone(G, n):
    # Keys that all score 0 and values of 0, but for one key whose weight is 2^-124 of the others' and whose
    # values are 1; ordinary values further in front.  The statistics do not depend on the values.
    L = 3000 + n
    b = make_batch([L], [n], num_kv_heads=1)
    q, k, v, _ = logical_tensors(b)
    q[:], k[:] = 0x4080, 0                           # 4 in every element
    k[2000] = synth.f32_to_bf16_bits(np.full(64, -2.6875, np.float32))   # -688 log2(e) / 8 = -124.07
    v[1000:2000], v[2000], v[2001:] = 0, 0x3F80, 0
    kc, vc = cpu_caches(b, k, v)
    mask = R.tree_masks([list(range(-1, n - 1))], 1)
    check(G, b, q, kc, vc, mask, None)
    # values at the lower end of bf16's normal range throughout, in that of fp32 as well
    q, k, v, sinks = logical_tensors(b)
    v = synth.f32_to_bf16_bits((synth.bf16_bits_to_f32(v) * np.float32(2.0 ** -124)).astype(np.float32))
    kc, vc = cpu_caches(b, k, v)
    check(G, b, q, kc, vc, mask, None)
    check(G, b, q, kc, vc, mask, sinks)
    # large ones as well
    v = synth.f32_to_bf16_bits((synth.bf16_bits_to_f32(v) * np.float32(2.0 ** 124) * np.float32(2.0 ** 44)).astype(np.float32))
    kc, vc = cpu_caches(b, k, v)
    check(G, b, q, kc, vc, mask, sinks)
    # and elements of very different size next to each other
    q, k, v, sinks = logical_tensors(b)
    v = synth.f32_to_bf16_bits(synth.bf16_bits_to_f32(v) * np.exp2(np.arange(64) % 13 * 2.0 + 10).astype(np.float32))
    kc, vc = cpu_caches(b, k, v)
    check(G, b, q, kc, vc, mask, sinks)


def rises_inside_ranges(b, q, kc, ks, tile):
    """Largest rise, in log2 units, of a row's scores inside one range above those of its first chunk."""
    heads, best = b.geom.num_kv_heads, 0.0
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    chunks = [(int(n) + 63) // 64 for n in b.seq_lens]
    tiles = [(int(n) + tile - 1) // tile for n in b.q_lens]
    total = sum(c * t for c, t in zip(chunks, tiles))
    per = max(-(-total // (2 * cus // heads)), 2)
    assert per >= 5
    at = 0
    for s in range(b.num_seqs):
        x, y, k = b.cu_seqlens_q[s], b.cu_seqlens_q[s + 1], R.cache_rows(b, kc, ks, s)
        plain = (int(b.seq_lens[s]) - int(y - x)) // 64          # chunks of context alone
        top = np.stack([(R.f64(q[x:y, h]) @ k[:plain * 64, h // 8].T).reshape(-1, plain, 64).max(2)
                        for h in range(8 * heads)], 2) * b.geom.softmax_scale * np.log2(np.e)
        for i in range(tiles[s]):
            for first in range(0, plain):
                if first and (at + first) % per:
                    continue                                     # (where a range begins)
                last = min(plain, first + per - (at + first) % per)
                best = max(best, float((top[tile * i:tile * i + tile, first:last] - top[tile * i:tile * i + tile, first:first + 1]).max()))
            at += chunks[s]
    return best


@pytest.mark.parametrize("kv_dtype", [KV_BF16, KV_FP8_E4M3])
@pytest.mark.parametrize("q_lens,tile", [([8, 5, 1], 8), ([16, 9, 12], 16), ([24, 20, 3], 24), ([30, 32, 17], 32), ([64, 40, 33], 32)])
def test_scores_that_outgrow_their_reference(G, q_lens, tile, kv_dtype):
    # A row's weights are taken relative to its range's first chunk until their sum reaches 2^60: the scores climb
    # by 75 log2 units from one chunk to the next, four times, and start again.  Scores of up to 320 log2 units whose
    # 64 products are off by 64 * 2^-24 * 320 = 1.2e-3 at most, twice that in the quotient: below the 2^-8 / 2 of
    # the bound; in lse, 1.2e-3 log2 units against 1e-5 * 220.
    lens = [8000, 7000, 9000]
    b = make_batch(lens, q_lens, num_kv_heads=8, kv_dtype=kv_dtype)
    q, k, v, sinks = logical_tensors(b)
    u = np.where(np.arange(64) % 3 == 0, 1.0, -0.5).astype(np.float32)
    t = np.concatenate([4.26 * (np.arange(n) // 64 % 5) for n in lens])
    q = synth.f32_to_bf16_bits((0.1 * synth.bf16_bits_to_f32(q) + 3.0 * u).astype(np.float32))
    k = synth.f32_to_bf16_bits((synth.bf16_bits_to_f32(k) + t[:, None, None] * u).astype(np.float32))
    ks, vs = fp8_scales(k, v) if kv_dtype == KV_FP8_E4M3 else (None, None)
    kc, vc = cpu_caches(b, k, v, ks, vs)
    assert rises_inside_ranges(b, q, kc, ks, tile) > 65
    rng = np.random.default_rng(1)
    mask = R.tree_masks([R.random_parents(n, rng) for n in q_lens], 1)
    for s in (sinks, None):
        check(G, b, q, kc, vc, mask, s, ks, vs)


@pytest.mark.parametrize("kv_dtype", [KV_BF16, KV_FP8_E4M3])
@pytest.mark.parametrize("seq_lens,q_lens", [([1], [1]), ([8, 9, 70], [8, 1, 7]), ([300, 65, 16, 17], [16, 9, 16, 1]),
                                             ([700, 64, 33], [33, 32, 17]), ([5000, 1100], [64, 63]), ([340, 256], [256, 200])])
@pytest.mark.parametrize("window", [0, 1, 7, 64, 200])
def test_random_trees_with_lse_and_without(G, seq_lens, q_lens, window, kv_dtype):
    b, q, kc, vc, ks, vs, sinks = R.filled(seq_lens, q_lens, window=window, kv_dtype=kv_dtype, num_kv_heads=2)
    rng = np.random.default_rng(window)
    words = (max(q_lens) + 63) // 64
    check(G, b, q, kc, vc, R.tree_masks([R.random_parents(n, rng, back=3) for n in q_lens], words), sinks, ks, vs)
    ints = [int.from_bytes(rng.bytes(8 * words), "little") for _ in range(sum(q_lens))]   # any set, bits behind q_len
    ints[0] = ints[-1] = 0
    for s in (sinks, None):
        check(G, b, q, kc, vc, R.masks_from_ints(ints, words), s, ks, vs)


def test_large_scores_without_lse(G):
    b, q, kc, vc, ks, vs, sinks = R.filled([900, 200], [6, 11], num_kv_heads=2)
    q = synth.f32_to_bf16_bits(synth.bf16_bits_to_f32(q) * 40)   # scores of hundreds: near one-hot rows
    rng = np.random.default_rng(4)
    mask = R.tree_masks([R.random_parents(n, rng) for n in (6, 11)], 1)
    for s in (sinks, np.full_like(sinks, 1e4), np.full_like(sinks, -np.inf)):
        check(G, b, q, kc, vc, mask, s)


@pytest.mark.parametrize("context", [60, 900])
def test_what_a_row_does_not_see_cannot_reach_it_without_lse(G, context):
    # drafted tokens with infinities and NaN in their keys and values; a whole span and a cut one
    b, q, kc, vc, ks, vs, sinks = R.filled([context + 6], [6], num_kv_heads=1)
    mask = R.masks_from_ints([0b1, 0b11, 0b101, 0b1011, 0b10101, 0b100001], 1)
    ref, _, mag = reference(b, q, kc, vc, mask, sinks)
    slots = b.all_slots(0)
    for bad in (0x7FC0, 0x7F80, 0xFF80):
        k2, v2 = kc.copy(), vc.copy()
        k2.reshape(-1, 1, 64)[slots[context + 2], 0, 3] = bad     # token 2: rows 2 and 4 see it
        v2.reshape(-1, 1, 64)[slots[context + 2], 0, 7] = bad
        v2.reshape(-1, 1, 64)[slots[context + 5], 0, 9] = bad     # token 5: row 5 alone
        out = ea.attn_tree(b.geom, G.bf16_dev(q), G.cache_dev(k2), G.cache_dev(v2), G.dev(b.block_table),
                           G.dev(b.seq_lens), G.dev(b.cu_seqlens_q), G.dev(mask), max_q_len=6, max_kv_len=b.max_kv_len,
                           sinks=G.dev(sinks))
        got, tol = R.f64(G.bits_host(out)), 3.5 * R.BF16_HALF_STEP * mag + 1e-6
        for i in (0, 1, 3):
            assert (np.abs(got[i] - ref[i]) <= tol[i]).all()
        rest = np.arange(64) != 9
        assert (np.abs(got[5] - ref[5]) <= tol[5])[:, rest].all() and not np.isfinite(got[5][:, 9]).any()
        assert not np.isfinite(got[2][:, 7]).all()
