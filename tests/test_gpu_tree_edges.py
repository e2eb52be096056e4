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
