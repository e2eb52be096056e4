"""eid_attn_tree against a plain 64-bit restatement.

Tolerance of an output element, with A = sum w |v| / sum w >= |out| computed beside the reference:
the weights of the numerator are rounded to bf16 (at most 2^-8 relative each, so at most 2^-8 A
together), the output once more (2^-8 |out|); the fp32 sums and exponentials stay below 2^-8 A / 2
(scores up to some hundreds: 2^-24 * 1000 relative).  So |error| <= 2.5 * 2^-8 A.  lse: fp32
throughout, a few 2^-24 of the scores and of the sum: |error| <= 1e-5 (1 + |lse|)."""
import numpy as np
import pytest
import torch

import eidola_amd as ea
from eidola_amd import KV_BF16, KV_FP8_E4M3

import cache_ref as R
from helpers import MAX_ABS_TOL

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def G():
    import gpu_helpers
    assert torch.cuda.is_available()
    ea.load_library()
    return gpu_helpers


def call(G, b, q, kc, vc, mask, sinks, ks=None, vs=None, **kw):
    kw.setdefault("max_q_len", b.max_q_len)
    kw.setdefault("max_kv_len", b.max_kv_len)
    return ea.attn_tree(b.geom, G.bf16_dev(q), G.cache_dev(kc), G.cache_dev(vc), G.dev(b.block_table),
                        G.dev(b.seq_lens), G.dev(b.cu_seqlens_q), G.dev(mask), sinks=G.dev(sinks), k_scale=G.dev(ks),
                        v_scale=G.dev(vs), return_lse=True, **kw)


def bound(b, q, kc, vc, mask, sinks, ks=None, vs=None):
    """sum of w |v| / sum of w for every output element."""
    mag = []
    for s in range(b.num_seqs):
        x, y = b.cu_seqlens_q[s], b.cu_seqlens_q[s + 1]
        see = R.tree_visible(mask[x:y], y - x, int(b.seq_lens[s]), b.geom.window)
        mag.append(R.attn_rows(R.f64(q[x:y]), R.cache_rows(b, kc, ks, s), np.abs(R.cache_rows(b, vc, vs, s)), see,
                               b.geom.softmax_scale, sinks)[0])
    return np.concatenate(mag)


def check(G, b, q, kc, vc, mask, sinks, ks=None, vs=None, **kw):
    out, lse = call(G, b, q, kc, vc, mask, sinks, ks, vs, **kw)
    ref, ref_lse = R.attn_tree(b, q, kc, vc, mask, sinks, ks, vs)
    got = R.f64(G.bits_host(out))
    assert np.isfinite(got).all()
    tol = 2.5 * R.BF16_HALF_STEP * bound(b, q, kc, vc, mask, sinks, ks, vs) + 1e-6
    assert (np.abs(got - ref) <= tol).all(), float((np.abs(got - ref) / tol).max())
    l = lse.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isinf(l), np.isinf(ref_lse))
    fine = np.isfinite(ref_lse)
    assert (np.abs(l[fine] - ref_lse[fine]) <= 1e-5 * (1 + np.abs(ref_lse[fine]))).all()
    return got


def trees(q_lens, seed, words=None):
    rng = np.random.default_rng(seed)
    return R.tree_masks([R.random_parents(n, rng) for n in q_lens], words or max(1, (max(q_lens) + 63) // 64))


@pytest.mark.parametrize("kv_dtype", [KV_BF16, KV_FP8_E4M3])
@pytest.mark.parametrize("seq_lens,q_lens", [
    ([1], [1]),                          # one token, no context
    ([8, 9, 70], [8, 1, 7]),             # a tree without context, beside others
    ([500, 37, 130], [8, 5, 3]),
    ([300, 65, 16, 17], [16, 9, 16, 1]),
    ([700, 64, 33], [33, 32, 17]),
    ([400, 1100], [64, 63]),             # two workgroups per tree
])
def test_random_trees(G, kv_dtype, seq_lens, q_lens):
    b, q, kc, vc, ks, vs, sinks = R.filled(seq_lens, q_lens, kv_dtype=kv_dtype, seed=3)
    check(G, b, q, kc, vc, trees(q_lens, 1), sinks, ks, vs)


@pytest.mark.parametrize("heads", [1, 2, 16])
def test_head_counts(G, heads):
    b, q, kc, vc, ks, vs, sinks = R.filled([150, 40], [10, 3], num_kv_heads=heads)
    check(G, b, q, kc, vc, trees([10, 3], 2), sinks)


@pytest.mark.parametrize("n", [65, 100, 128, 200, 256])
def test_masks_of_several_words(G, n):
    b, q, kc, vc, ks, vs, sinks = R.filled([n + 77], [n], num_kv_heads=1)
    check(G, b, q, kc, vc, trees([n], n), sinks)
    check(G, b, q, kc, vc, trees([n], n, words=4), None)


@pytest.mark.parametrize("window", [1, 2, 5, 17, 64, 128, 100000])
@pytest.mark.parametrize("kv_dtype", [KV_BF16, KV_FP8_E4M3])
def test_windows_are_measured_in_depths(G, window, kv_dtype):
    seq_lens, q_lens = [400, 60, 40, 9], [40, 12, 1, 9]
    b, q, kc, vc, ks, vs, sinks = R.filled(seq_lens, q_lens, window=window, kv_dtype=kv_dtype, num_kv_heads=2)
    rng = np.random.default_rng(window)
    mask = R.tree_masks([R.random_parents(n, rng, back=2) for n in q_lens], 1)   # deep trees
    check(G, b, q, kc, vc, mask, sinks, ks, vs)


def test_long_contexts_are_cut_and_joined(G):
    # ranges that end inside sequences: many pieces for one row, and pieces of neighbours in one range
    seq_lens, q_lens = [9000, 65, 3000, 20, 4097], [5, 8, 1, 2, 7]
    b, q, kc, vc, ks, vs, sinks = R.filled(seq_lens, q_lens, num_kv_heads=1, seed=9)
    mask = trees(q_lens, 5)
    got = check(G, b, q, kc, vc, mask, sinks)
    again = check(G, b, q, kc, vc, mask, sinks, sum_kv_len=int(b.seq_lens.sum()))
    assert np.abs(got - again).max() <= MAX_ABS_TOL
    check(G, b, q, kc, vc, mask, None, max_q_len=20, max_kv_len=9007)   # bounds above the truth


def test_chain_equals_the_ragged_call(G):
    # a tree without branches is what eid_attn_varlen computes
    seq_lens, q_lens = [333, 1000, 64], [5, 20, 40]
    for window in (0, 128):
        b, q, kc, vc, ks, vs, sinks = R.filled(seq_lens, q_lens, window=window)
        mask = R.tree_masks([list(range(-1, n - 1)) for n in q_lens], 1)
        got = check(G, b, q, kc, vc, mask, sinks)
        line = R.f64(G.run_attn(b, q, G.cache_dev(kc), G.cache_dev(vc), sinks))
        assert np.abs(got - line).max() <= MAX_ABS_TOL


@pytest.mark.parametrize("with_sinks", [True, False])
@pytest.mark.parametrize("window", [0, 3])
def test_rows_that_see_nothing_and_arbitrary_masks(G, with_sinks, window):
    seq_lens, q_lens = [12, 90, 70], [12, 20, 6]
    b, q, kc, vc, ks, vs, sinks = R.filled(seq_lens, q_lens, window=window, num_kv_heads=1)
    rng = np.random.default_rng(0)
    ints = [int(x) for x in rng.integers(0, 1 << 62, sum(q_lens))]      # bits beyond q_len among them
    ints[0] = ints[5] = 0                                                # no context, no bit: nothing to see
    ints[12] = 0                                                         # context only
    ints[13] = (1 << 64) - 1
    mask = R.masks_from_ints(ints, 1)
    got = check(G, b, q, kc, vc, mask, sinks if with_sinks else None)
    assert (got[0] == 0).all() and (got[5] == 0).all()


def test_what_a_row_does_not_see_cannot_reach_it(G):
    # siblings with infinities and NaN in their keys and values, rows of no sequence, unwritten rows
    # behind the end (the caches start out as NaN)
    b, q, kc, vc, ks, vs, sinks = R.filled([100], [6], num_kv_heads=1)
    mask = R.masks_from_ints([0b1, 0b11, 0b101, 0b1011, 0b10101, 0b100001], 1)
    ref, _ = R.attn_tree(b, q, kc, vc, mask, sinks)
    slots = b.all_slots(0)
    for bad in (0x7FC0, 0x7F80, 0xFF80):
        k2, v2 = kc.copy(), vc.copy()
        k2.reshape(-1, 1, 64)[slots[96], 0, 3] = bad     # token 2: rows 2 and 4 see it
        v2.reshape(-1, 1, 64)[slots[96], 0, 7] = bad
        v2.reshape(-1, 1, 64)[slots[99], 0, :] = bad     # token 5: row 5 alone
        out = R.f64(G.bits_host(call(G, b, q, k2, v2, mask, sinks)[0]))
        for i in (0, 1, 3):
            assert np.abs(out[i] - ref[i]).max() <= MAX_ABS_TOL
        assert not np.isfinite(out[5]).any()
        assert not np.isfinite(out[2][:, 7]).all()


def test_a_visible_infinity_stays_in_its_column(G):
    b, q, kc, vc, ks, vs, sinks = R.filled([80], [3], num_kv_heads=1)
    mask = R.masks_from_ints([0b1, 0b11, 0b101], 1)
    ref, _ = R.attn_tree(b, q, kc, vc, mask, sinks)
    vc.reshape(-1, 1, 64)[b.all_slots(0)[78], 0, 9] = 0x7F80     # +inf in token 1: row 1 alone
    out = R.f64(G.bits_host(call(G, b, q, kc, vc, mask, sinks)[0]))
    assert (out[1][:, 9] == np.inf).all()
    out[1][:, 9] = ref[1][:, 9]
    assert np.abs(out - ref).max() <= MAX_ABS_TOL


def test_large_scores(G):
    b, q, kc, vc, ks, vs, sinks = R.filled([900, 200], [6, 11], num_kv_heads=2)
    from eidola_amd import synth
    q = synth.f32_to_bf16_bits(synth.bf16_bits_to_f32(q) * 40)   # scores of hundreds: near one-hot rows
    check(G, b, q, kc, vc, trees([6, 11], 4), sinks)
    check(G, b, q, kc, vc, trees([6, 11], 4), np.full_like(sinks, 1e4))
    check(G, b, q, kc, vc, trees([6, 11], 4), np.full_like(sinks, -np.inf))


def test_rows_of_no_sequence_stay_and_empty_sequences_are_skipped(G):
    b, q, kc, vc, ks, vs, sinks = R.filled([50, 30], [4, 2], num_kv_heads=1)
    mask = trees([4, 2], 7)
    ref, _ = R.attn_tree(b, q, kc, vc, mask, sinks)
    # three sequences, the middle one without rows; two rows of padding behind the last
    cu = np.array([0, 4, 4, 6], np.int32)
    lens = np.array([50, 0, 30], np.int32)
    bt = np.stack([b.block_table[0], np.full_like(b.block_table[0], 10 ** 6), b.block_table[1]])   # junk ids
    pad = np.concatenate([q, q[:2]])
    out = torch.full((8, 8, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    ea.attn_tree(b.geom, G.bf16_dev(pad), G.cache_dev(kc), G.cache_dev(vc), G.dev(bt), G.dev(lens), G.dev(cu),
                 G.dev(np.concatenate([mask, mask[:2]])), sinks=G.dev(sinks), max_q_len=4, max_kv_len=50, out=out)
    got = R.f64(G.bits_host(out))
    assert np.abs(got[:6] - ref).max() <= MAX_ABS_TOL and (got[6:] == 7).all()


def test_captured_once_serves_other_lengths_and_masks(G):
    b, q, kc, vc, ks, vs, sinks = R.filled([300, 90], [6, 4], num_kv_heads=2)
    masks = [trees([6, 4], s) for s in (1, 2, 3)]
    lens = [np.array([300, 90]), np.array([250, 61]), np.array([99, 7])]
    g = b.geom
    lens_d, mask_d = G.dev(lens[0].astype(np.int32)), G.dev(masks[0])
    q_d, k_d, v_d, bt, cu = G.bf16_dev(q), G.cache_dev(kc), G.cache_dev(vc), G.dev(b.block_table), G.dev(b.cu_seqlens_q)
    s_d = G.dev(sinks)
    out = torch.empty_like(q_d)
    desc = ea.make_desc(g, num_seqs=2, num_q_tokens=10, max_q_len=6, max_kv_len=300, max_blocks_per_seq=bt.shape[1],
                        num_blocks=k_d.shape[0])
    ws = torch.empty(ea.attn_tree_workspace_bytes(desc), dtype=torch.uint8, device="cuda")
    run = lambda: ea.attn_tree(g, q_d, k_d, v_d, bt, lens_d, cu, mask_d, sinks=s_d, max_q_len=6, max_kv_len=300,
                               out=out, workspace=ws)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    from eidola_amd import synth
    for turn in range(4):
        m, n = masks[turn % 3], lens[turn % 3].astype(np.int32)
        lens_d.copy_(G.dev(n))
        mask_d.copy_(G.dev(m))
        out.zero_()
        ws.fill_(255)                       # nothing in the workspace has to start from a value
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = G.bits_host(out)
        b2 = synth.Batch("other", g, n, b.q_lens, b.block_table, b.num_blocks, b.seed)
        ref, _ = R.attn_tree(b2, q, kc, vc, m, sinks)
        assert np.abs(R.f64(got) - ref).max() <= MAX_ABS_TOL
        run()
        assert np.array_equal(got, G.bits_host(out))


def test_another_stream_and_the_same_bits(G):
    b, q, kc, vc, ks, vs, sinks = R.filled([2000, 700], [12, 30])
    mask = trees([12, 30], 8)
    first = G.bits_host(call(G, b, q, kc, vc, mask, sinks)[0])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = call(G, b, q, kc, vc, mask, sinks)[0]
    side.synchronize()
    assert np.array_equal(first, G.bits_host(second))


def test_a_page_past_two_to_the_32_bytes(G):
    # pages at the far end of a cache whose byte offsets do not fit 32 bits (4.3 GB per tensor)
    nb = (1 << 32) // 16384 + 40
    b, q, kc, vc, ks, vs, sinks = R.filled([100, 60], [5, 3])
    mask = trees([5, 3], 6)
    ref, _ = R.attn_tree(b, q, kc, vc, mask, sinks)
    big = [torch.zeros((nb, 16, 8, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for t, c in zip(big, (kc, vc)):
        t[nb - kc.shape[0]:] = G.cache_dev(c)
    bt = b.block_table + (nb - kc.shape[0])
    out = ea.attn_tree(b.geom, G.bf16_dev(q), big[0], big[1], G.dev(bt.astype(np.int32)), G.dev(b.seq_lens),
                       G.dev(b.cu_seqlens_q), G.dev(mask), sinks=G.dev(sinks), max_q_len=5, max_kv_len=100)
    assert np.abs(R.f64(G.bits_host(out)) - ref).max() <= MAX_ABS_TOL


@pytest.mark.parametrize("kv_dtype", [KV_BF16, KV_FP8_E4M3])
@pytest.mark.parametrize("q_lens", [[5, 1], [16, 9], [24, 20], [40, 64]])
def test_scores_that_rise_along_the_context(G, q_lens, kv_dtype):
    # every row's scores climb along the context, by 14 log2 units from 64 keys to the next, and fall again
    # behind its third quarter, so that the reference of a row's weights has to follow.  Scores of up to 245
    # log2 units whose 64 products have one sign: off by at most 64 * 2^-24 * 245 = 9.4e-4, twice that in
    # the quotient: below the 2^-8 / 2 of the bound.
    from eidola_amd import synth
    from helpers import cpu_caches, fp8_scales, logical_tensors, make_batch
    b = make_batch([1500, 400], q_lens, num_kv_heads=2, kv_dtype=kv_dtype)
    q, k, v, sinks = logical_tensors(b)
    u = np.where(np.arange(64) % 3 == 0, 1.0, -0.5).astype(np.float32)
    t = np.concatenate([np.minimum(np.arange(n), 1.5 * n - np.arange(n)) / 80.0 for n in b.seq_lens])
    q = synth.f32_to_bf16_bits((0.25 * synth.bf16_bits_to_f32(q) + 3.0 * u).astype(np.float32))
    k = synth.f32_to_bf16_bits((synth.bf16_bits_to_f32(k) + t[:, None, None] * u).astype(np.float32))
    ks, vs = fp8_scales(k, v) if b.geom.kv_dtype == KV_FP8_E4M3 else (None, None)
    kc, vc = cpu_caches(b, k, v, ks, vs)
    mask = trees(q_lens, 21)
    for s in (sinks, np.full_like(sinks, -np.inf)):
        check(G, b, q, kc, vc, mask, s, ks, vs)
    # the call without lse sums its weights in another way
    got = ea.attn_tree(b.geom, G.bf16_dev(q), G.cache_dev(kc), G.cache_dev(vc), G.dev(b.block_table),
                       G.dev(b.seq_lens), G.dev(b.cu_seqlens_q), G.dev(mask), k_scale=G.dev(ks), v_scale=G.dev(vs),
                       max_q_len=b.max_q_len, max_kv_len=b.max_kv_len)
    ref, _ = R.attn_tree(b, q, kc, vc, mask, None, ks, vs)
    tol = 2.5 * R.BF16_HALF_STEP * bound(b, q, kc, vc, mask, None, ks, vs) + 1e-6
    assert (np.abs(R.f64(G.bits_host(got)) - ref) <= tol).all()


@pytest.mark.parametrize("lens,q_lens", [([3000, 700], [6, 4]), ([2500, 64], [30, 64]), ([900, 200], [200, 100])])
def test_captured_with_contexts_that_are_cut(G, lens, q_lens):
    b, q, kc, vc, ks, vs, sinks = R.filled(lens, q_lens, num_kv_heads=2)
    from eidola_amd import synth
    g = b.geom
    words = (max(q_lens) + 63) // 64
    masks = [trees(q_lens, s, words) for s in (1, 2)]
    lens_d, mask_d = G.dev(b.seq_lens), G.dev(masks[0])
    q_d, k_d, v_d, bt, cu = G.bf16_dev(q), G.cache_dev(kc), G.cache_dev(vc), G.dev(b.block_table), G.dev(b.cu_seqlens_q)
    out = torch.empty_like(q_d)
    desc = ea.make_desc(g, num_seqs=2, num_q_tokens=len(q), max_q_len=max(q_lens), max_kv_len=lens[0],
                        max_blocks_per_seq=bt.shape[1], num_blocks=k_d.shape[0])
    ws = torch.empty(ea.attn_tree_workspace_bytes(desc), dtype=torch.uint8, device="cuda")
    run = lambda: ea.attn_tree(g, q_d, k_d, v_d, bt, lens_d, cu, mask_d, max_q_len=max(q_lens), max_kv_len=lens[0],
                               out=out, workspace=ws)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for turn in range(4):
        n = np.array([[lens[0], lens[1]], [lens[1], lens[1]], [q_lens[0], lens[1]], [lens[0] - 77, q_lens[1]]][turn],
                     np.int32)
        n = np.maximum(n, np.array(q_lens, np.int32))
        m = masks[turn % 2]
        lens_d.copy_(G.dev(n))
        mask_d.copy_(G.dev(m))
        out.zero_()
        ws.fill_(255)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = G.bits_host(out)
        b2 = synth.Batch("other", g, n, b.q_lens, b.block_table, b.num_blocks, b.seed)
        ref, _ = R.attn_tree(b2, q, kc, vc, m, None)
        tol = 2.5 * R.BF16_HALF_STEP * bound(b2, q, kc, vc, m, None) + 1e-6
        assert (np.abs(R.f64(got) - ref) <= tol).all()
        run()
        assert np.array_equal(got, G.bits_host(out))


@pytest.mark.parametrize("kv_dtype", [KV_BF16, KV_FP8_E4M3])
@pytest.mark.parametrize("heads", [4, 24])
def test_other_head_counts(G, heads, kv_dtype):
    q_lens = [9, 30]
    b, q, kc, vc, ks, vs, sinks = R.filled([700, 90], q_lens, num_kv_heads=heads, kv_dtype=kv_dtype)
    check(G, b, q, kc, vc, trees(q_lens, 5), sinks, ks, vs)
