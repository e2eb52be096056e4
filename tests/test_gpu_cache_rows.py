"""eid_kv_score, eid_kv_select and eid_kv_compact against plain 64-bit restatements.

Scores: a term e^(s - lse) has an exponent of at most 64 in log2 units, computed in fp32 with three
roundings (3 * 2^-24 * 64 = 1.2e-5) from a score whose 64 products are summed in fp32 (64 * 2^-24
of the sum of their magnitudes, about 6: 2.3e-5 at most); n terms are added (n 2^-24 = 2.4e-5 for
the n <= 400 here).  Together at most 6e-5 of the sum; 1e-7 beside it for sums that vanish.
Selections and moves are exact."""
import numpy as np
import pytest
import torch

import eidola_amd as ea
from eidola_amd import KV_BF16, KV_FP8_E4M3

import cache_ref as R

pytestmark = pytest.mark.gpu
REL = 6e-5


@pytest.fixture(scope="module")
def G():
    import gpu_helpers
    assert torch.cuda.is_available()
    ea.load_library()
    return gpu_helpers


def lse_of(b, q, kc, vc, sinks, ks, vs):
    """The attention call's lse in 64 bits, as fp32."""
    mask = R.tree_masks([list(range(-1, int(n) - 1)) for n in b.q_lens], (b.max_q_len + 63) // 64)
    return R.attn_tree(b, q, kc, vc, mask, sinks, ks, vs)[1].astype(np.float32)


def pool(b, rng):
    w = rng.random((b.num_blocks, b.geom.num_kv_heads, 16)).astype(np.float32)
    return w


def score(G, b, q, lse, kc, w, ks=None, **kw):
    kw.setdefault("max_q_len", b.max_q_len)
    kw.setdefault("max_kv_len", b.max_kv_len)
    return ea.kv_score(b.geom, G.bf16_dev(q), G.dev(lse), G.cache_dev(kc), G.dev(b.block_table), G.dev(b.seq_lens),
                       G.dev(b.cu_seqlens_q), G.dev(w), k_scale=G.dev(ks), **kw).cpu().numpy()


@pytest.mark.parametrize("kv_dtype", [KV_BF16, KV_FP8_E4M3])
@pytest.mark.parametrize("window", [0, 1, 20])
@pytest.mark.parametrize("seq_lens,q_lens", [
    ([1], [1]), ([17, 300, 64], [1, 1, 1]), ([2, 33, 200], [2, 1, 2]), ([3, 130], [3, 50]),
    ([200, 129, 40, 16], [37, 1, 2, 16]), ([128, 150], [128, 33]),
])
def test_scores(G, kv_dtype, window, seq_lens, q_lens):
    b, q, kc, vc, ks, vs, sinks = R.filled(seq_lens, q_lens, kv_dtype=kv_dtype, window=window, num_kv_heads=2)
    lse = lse_of(b, q, kc, vc, sinks, ks, vs)
    w = pool(b, np.random.default_rng(1))
    got, ref = score(G, b, q, lse, kc, w, ks), R.kv_score(b, q, lse, kc, w, ks)
    assert (np.abs(got - ref) <= REL * ref + 1e-7).all(), float((np.abs(got - ref) / (ref + 1e-9)).max())
    used = np.zeros(w.shape, bool)
    s = np.concatenate([b.all_slots(i) for i in range(b.num_seqs)])
    used[s // 16, :, s % 16] = True
    assert np.array_equal(got[~used], w[~used])        # rows of no sequence stay as they were
    assert np.array_equal(got, score(G, b, q, lse, kc, w, ks, max_q_len=b.max_q_len + 0,
                                     sum_kv_len=int(b.seq_lens.sum())))


@pytest.mark.parametrize("heads", [1, 8, 16])
def test_score_head_counts(G, heads):
    for q_lens in ([1, 1], [9, 1]):
        b, q, kc, vc, ks, vs, sinks = R.filled([90, 40], q_lens, num_kv_heads=heads)
        lse = lse_of(b, q, kc, vc, None, ks, vs)
        w = pool(b, np.random.default_rng(2))
        ref = R.kv_score(b, q, lse, kc, w)
        assert (np.abs(score(G, b, q, lse, kc, w) - ref) <= REL * ref + 1e-7).all()


def test_weights_of_a_row_add_up_to_one_less_its_sink(G):
    b, q, kc, vc, ks, vs, sinks = R.filled([700, 90], [1, 60])
    bt, sl, cu = G.dev(b.block_table), G.dev(b.seq_lens), G.dev(b.cu_seqlens_q)
    out, lse = ea.attn_varlen(b.geom, G.bf16_dev(q), G.cache_dev(kc), G.cache_dev(vc), bt, sl, cu, max_q_len=60,
                              max_kv_len=700, sinks=G.dev(sinks), return_lse=True)
    w = np.full((b.num_blocks, 8, 16), 0.0, np.float32)
    got = score(G, b, q, lse.cpu().numpy(), kc, w).astype(np.float64)
    share = 1 - np.exp(sinks[None, :] - lse.cpu().numpy().astype(np.float64))     # [T, Hq]
    for s in range(2):
        sl_ = b.all_slots(s)
        a, e = b.cu_seqlens_q[s], b.cu_seqlens_q[s + 1]
        total = got[sl_ // 16, :, sl_ % 16].sum(0)
        assert np.allclose(total, share[a:e].reshape(-1, 8, 8).sum((0, 2)), rtol=1e-4)


def test_rows_that_saw_nothing_add_nothing_and_new_keys_start_from_zero(G):
    b, q, kc, vc, ks, vs, sinks = R.filled([40, 20], [1, 5], num_kv_heads=1)
    lse = lse_of(b, q, kc, vc, None, ks, vs)
    lse[0], lse[2] = -np.inf, -np.inf
    w = np.full((b.num_blocks, 1, 16), np.nan, np.float32)       # a page's last owner left junk
    got = score(G, b, q, lse, kc, w)
    s0, s1 = b.all_slots(0), b.all_slots(1)
    assert got[s0[39] // 16, 0, s0[39] % 16] == 0
    assert np.isfinite(got[s1[15:] // 16, 0, s1[15:] % 16]).all()
    assert np.isnan(got[s0[:39] // 16, 0, s0[:39] % 16]).all()


def test_score_skips_empty_sequences_and_junk_pages(G):
    b, q, kc, vc, ks, vs, sinks = R.filled([50, 30], [4, 1], num_kv_heads=1)
    lse = lse_of(b, q, kc, vc, sinks, ks, vs)
    w = pool(b, np.random.default_rng(3))
    ref = R.kv_score(b, q, lse, kc, w)
    bt = np.stack([b.block_table[0], np.full_like(b.block_table[0], -7), b.block_table[1]])
    got = ea.kv_score(b.geom, G.bf16_dev(q), G.dev(lse), G.cache_dev(kc), G.dev(bt),
                      G.dev(np.array([50, 0, 30], np.int32)), G.dev(np.array([0, 4, 4, 5], np.int32)), G.dev(w),
                      max_q_len=4, max_kv_len=50).cpu().numpy()
    assert (np.abs(got - ref) <= REL * ref + 1e-7).all()


# ---- selection ---------------------------------------------------------------------------------

def select(G, b, w, budget, first, last, **kw):
    keep, counts = ea.kv_select(b.geom, G.dev(w), G.dev(b.block_table), G.dev(b.seq_lens), budget=budget,
                                keep_first=first, keep_last=last, max_kv_len=b.max_kv_len, **kw)
    return keep.cpu().numpy(), counts.cpu().numpy()


def kinds(rng, shape):
    yield rng.random(shape).astype(np.float32)
    yield (rng.integers(0, 4, shape) / 4).astype(np.float32)                       # ties everywhere
    yield np.zeros(shape, np.float32)                                              # nothing but ties
    yield np.where(rng.random(shape) < 0.5, -0.0, 0.0).astype(np.float32)          # both zeros are one value
    x = rng.standard_normal(shape).astype(np.float32) * 10.0 ** rng.integers(-30, 30, shape).astype(np.float32)
    for v in (np.nan, np.inf, -np.inf, 1e-45, -1e-45):
        x[rng.random(shape) < 0.1] = v
    yield x
    yield (1.0 + rng.integers(0, 300, shape) * 2.0 ** -23).astype(np.float32)       # the last bits decide


@pytest.mark.parametrize("seq_lens,budget,first,last", [
    ([1, 16, 17, 40], 16, 0, 0), ([40, 41, 100, 39], 40, 4, 16), ([300, 64, 1500], 64, 64, 0),
    ([300, 65, 1500], 64, 0, 64), ([2500, 5], 1, 0, 0), ([2500, 700, 4100], 699, 3, 7),
    ([5000, 1025, 1024], 1024, 1, 1), ([600, 90], 50, 20, 30),
])
def test_selection(G, seq_lens, budget, first, last):
    b = R.make_batch(seq_lens, [1] * len(seq_lens), num_kv_heads=2)
    rng = np.random.default_rng(budget)
    for w in kinds(rng, (b.num_blocks, 2, 16)):
        keep, counts = select(G, b, w, budget, first, last)
        ref, ref_counts = R.kv_select(b, w, budget, first, last)
        assert np.array_equal(counts, ref_counts) and np.array_equal(keep, ref)


@pytest.mark.parametrize("length", [8191, 32768, 70001])
def test_selection_of_long_sequences(G, length):
    b = R.make_batch([length], [1], num_kv_heads=1)
    rng = np.random.default_rng(length)
    for w in (rng.random((b.num_blocks, 1, 16)).astype(np.float32),
              (rng.integers(0, 9, (b.num_blocks, 1, 16))).astype(np.float32)):
        keep, _ = select(G, b, w, length // 3, 4, 32)
        assert np.array_equal(keep, R.kv_select(b, w, length // 3, 4, 32)[0])


# ---- moves -------------------------------------------------------------------------------------

def layer_caches(b, n, seed):
    rng = np.random.default_rng(seed)
    shape = (b.num_blocks, 16, b.geom.num_kv_heads, 64)
    if b.geom.kv_dtype == KV_FP8_E4M3:
        return [rng.integers(0, 256, shape).astype(np.uint8) for _ in range(n)]
    return [rng.integers(0, 65536, shape).astype(np.uint16) for _ in range(n)]


@pytest.mark.parametrize("kv_dtype", [KV_BF16, KV_FP8_E4M3])
@pytest.mark.parametrize("heads", [1, 2, 8, 16])
def test_accepted_paths_move_in_every_layer(G, kv_dtype, heads):
    b = R.make_batch([60, 17, 200, 9], [1] * 4, num_kv_heads=heads, kv_dtype=kv_dtype)
    starts = np.array([40, 16, 190, 0], np.int32)
    rows = [[40, 43, 44, 59], [16], [191, 193, 195, 197, 199], [2, 4, 8]]
    keep = np.full((4, 6), -1, np.int32)
    for s, r in enumerate(rows):
        keep[s, :len(r)] = r
    counts = np.array([len(r) for r in rows], np.int32)
    ks, vs = layer_caches(b, 3, 1), layer_caches(b, 3, 2)
    kd, vd = [G.cache_dev(c) for c in ks], [G.cache_dev(c) for c in vs]
    ea.kv_compact(b.geom, kd, vd, G.dev(b.block_table), G.dev(b.seq_lens), G.dev(keep), G.dev(counts),
                  starts=G.dev(starts))
    for host, dev in zip(ks + vs, kd + vd):
        assert np.array_equal(G.cache_host(dev), R.kv_compact(b, host, keep, counts, starts, False))


@pytest.mark.parametrize("kv_dtype", [KV_BF16, KV_FP8_E4M3])
@pytest.mark.parametrize("heads,layers", [(1, 1), (8, 2), (2, 70)])
def test_rows_kept_per_head_move_with_their_scores(G, kv_dtype, heads, layers):
    seq_lens = [700, 33, 129, 1] if layers < 70 else [90, 33]
    b = R.make_batch(seq_lens, [1] * len(seq_lens), num_kv_heads=heads, kv_dtype=kv_dtype)
    rng = np.random.default_rng(heads)
    N = 300
    keep = np.full((layers, b.num_seqs, heads, N), -1, np.int32)
    counts = np.minimum(b.seq_lens, [250, 20, 129, 1][:b.num_seqs]).astype(np.int32)
    for l in range(layers):
        for s in range(b.num_seqs):
            for h in range(heads):
                keep[l, s, h, :counts[s]] = np.sort(rng.permutation(int(b.seq_lens[s]))[:counts[s]])
    ks, vs = layer_caches(b, layers, 3), layer_caches(b, layers, 4)
    ws = [rng.random((b.num_blocks, heads, 16)).astype(np.float32) for _ in range(layers)]
    kd, vd, wd = [G.cache_dev(c) for c in ks], [G.cache_dev(c) for c in vs], [G.dev(w) for w in ws]
    ea.kv_compact(b.geom, kd, vd, G.dev(b.block_table), G.dev(b.seq_lens), G.dev(keep), G.dev(counts), scores=wd)
    zero = np.zeros(b.num_seqs, int)
    for l in range(layers):
        for host, dev in ((ks[l], kd[l]), (vs[l], vd[l])):
            assert np.array_equal(G.cache_host(dev), R.kv_compact(b, host, keep[l], counts, zero, True))
        moved = R.kv_compact(b, np.ascontiguousarray(ws[l].transpose(0, 2, 1)), keep[l], counts, zero, True)
        assert np.array_equal(wd[l].cpu().numpy(), moved.transpose(0, 2, 1))


@pytest.mark.parametrize("kv_dtype", [KV_BF16, KV_FP8_E4M3])
def test_long_moves_in_place(G, kv_dtype):
    # several steps of the largest workgroup, and rows that move by one (the closest a move comes
    # to what it has yet to read)
    L = 6000
    b = R.make_batch([L], [1], num_kv_heads=1, kv_dtype=kv_dtype)
    for rows in (np.arange(1, L), np.arange(0, L, 2), np.concatenate([np.arange(4), np.arange(L - 3500, L)])):
        keep, counts = rows.astype(np.int32)[None, None], np.array([len(rows)], np.int32)
        ks, vs = layer_caches(b, 1, 5), layer_caches(b, 1, 6)
        kd, vd = G.cache_dev(ks[0]), G.cache_dev(vs[0])
        ea.kv_compact(b.geom, [kd], [vd], G.dev(b.block_table), G.dev(b.seq_lens), G.dev(keep), G.dev(counts))
        for host, dev in ((ks[0], kd), (vs[0], vd)):
            assert np.array_equal(G.cache_host(dev), R.kv_compact(b, host, keep, counts, [0], True))


def test_entries_that_may_not_move_do_not(G):
    # before their place, behind the end, negative; counts beyond the list; starts behind the end
    b = R.make_batch([20, 20, 20], [1] * 3, num_kv_heads=1)
    keep = np.array([[3, 2, 19, 25, -4], [10 ** 9, 0, 5, 6, 7], [1, 2, 3, 4, 5]], np.int32)
    counts, starts = np.array([5, 90, 3], np.int32), np.array([2, 0, 10 ** 6], np.int32)
    ks, vs = layer_caches(b, 1, 7), layer_caches(b, 1, 8)
    kd, vd = G.cache_dev(ks[0]), G.cache_dev(vs[0])
    ea.kv_compact(b.geom, [kd], [vd], G.dev(b.block_table), G.dev(b.seq_lens), G.dev(keep), G.dev(counts),
                  starts=G.dev(starts))
    for host, dev in ((ks[0], kd), (vs[0], vd)):
        ref = host.copy().reshape(-1, 1, 64)
        old, s = host.reshape(-1, 1, 64), [b.all_slots(i) for i in range(3)]
        ref[s[0][2]], ref[s[0][4]] = old[s[0][3]], old[s[0][19]]
        for i, r in ((2, 5), (3, 6), (4, 7)):
            ref[s[1][i]] = old[s[1][r]]
        assert np.array_equal(G.cache_host(dev), ref.reshape(host.shape))


def test_captured_selection_and_move_serve_other_lengths(G):
    b = R.make_batch([400, 150], [1, 1], num_kv_heads=2)
    rng = np.random.default_rng(1)
    w = rng.random((b.num_blocks, 2, 16)).astype(np.float32)
    w_d, bt, lens_d = G.dev(w), G.dev(b.block_table), G.dev(b.seq_lens)
    ks, vs = layer_caches(b, 1, 9)[0], layer_caches(b, 1, 10)[0]
    kd, vd = G.cache_dev(ks), G.cache_dev(vs)
    keep = torch.empty((2, 2, 100), dtype=torch.int32, device="cuda")
    counts = torch.empty(2, dtype=torch.int32, device="cuda")

    def run():
        ea.kv_select(b.geom, w_d, bt, lens_d, budget=100, keep_first=4, keep_last=8, max_kv_len=400, keep=keep,
                     counts=counts)
        ea.kv_compact(b.geom, [kd], [vd], bt, lens_d, keep, counts, scores=[w_d])
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    from eidola_amd import synth
    for lens in ([400, 150], [399, 90], [101, 130], [400, 1]):
        n = np.array(lens, np.int32)
        lens_d.copy_(G.dev(n))
        w_d.copy_(G.dev(w))
        kd.copy_(G.cache_dev(ks))
        vd.copy_(G.cache_dev(vs))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        b2 = synth.Batch("other", b.geom, n, b.q_lens, b.block_table, b.num_blocks, b.seed)
        rk, rc = R.kv_select(b2, w, 100, 4, 8)
        assert np.array_equal(keep.cpu().numpy(), rk) and np.array_equal(counts.cpu().numpy(), rc)
        assert np.array_equal(G.cache_host(kd), R.kv_compact(b2, ks, rk, rc, [0, 0], True))
        assert np.array_equal(G.cache_host(vd), R.kv_compact(b2, vs, rk, rc, [0, 0], True))


@pytest.mark.parametrize("kv_dtype", [KV_BF16, KV_FP8_E4M3])
@pytest.mark.parametrize("heads,window", [(8, 0), (8, 100), (16, 0), (16, 33)])
def test_scores_of_many_sequences(G, heads, window, kv_dtype):
    # more sequences than lanes, some of more rows than the single-token kernel takes, some of one chunk
    rng = np.random.default_rng(heads + window)
    q_lens = [int(n) for n in rng.choice([1, 1, 1, 2, 2, 5], 90)]
    seq_lens = [int(rng.choice([n, 63, 64, 65, 128, int(rng.integers(n, 500))])) for n in q_lens]
    seq_lens[40], q_lens[40] = 3000, 1
    b, q, kc, vc, ks, vs, sinks = R.filled(seq_lens, q_lens, num_kv_heads=heads, window=window, kv_dtype=kv_dtype)
    lse = lse_of(b, q, kc, vc, sinks, ks, vs)
    w = pool(b, rng)
    ref = R.kv_score(b, q, lse, kc, w, ks)
    for kw in ({}, dict(sum_kv_len=int(b.seq_lens.sum())), dict(max_kv_len=3008)):
        got = score(G, b, q, lse, kc, w, ks, **kw)
        assert (np.abs(got - ref) <= REL * ref + 1e-7).all()


@pytest.mark.parametrize("heads", [2, 8])
def test_a_padded_batch_may_hold_sequences_of_few_rows(G, heads):
    # as many tokens as sequences x max_q_len, the sequences themselves shorter: rows of padding behind them
    b, q, kc, vc, ks, vs, sinks = R.filled([90, 700, 64], [1, 6, 2], num_kv_heads=heads)
    lse = lse_of(b, q, kc, vc, sinks, ks, vs)
    w = pool(b, np.random.default_rng(6))
    ref = R.kv_score(b, q, lse, kc, w)
    q2, lse2 = np.concatenate([q, q]), np.concatenate([lse, lse])
    assert len(q2) == 3 * b.max_q_len
    got = score(G, b, q2, lse2, kc, w)
    assert (np.abs(got - ref) <= REL * ref + 1e-7).all()


def test_captured_scores_serve_other_lengths(G):
    for q_lens in ([1, 2, 1], [70, 3, 1]):
        b, q, kc, vc, ks, vs, sinks = R.filled([700, 1200, 300], q_lens)
        w = pool(b, np.random.default_rng(4))
        cases = []
        from eidola_amd import synth
        for lens in (b.seq_lens, np.array([90, 1190, 65]), np.array([70, 600, 1])):
            n = np.array(lens, np.int32)
            b2 = synth.Batch("other", b.geom, n, b.q_lens, b.block_table, b.num_blocks, b.seed)
            lse = lse_of(b2, q, kc, vc, sinks, ks, vs)
            cases.append((n, lse, R.kv_score(b2, q, lse, kc, w)))
        w_d, lens_d, lse_d = G.dev(w), G.dev(b.seq_lens), G.dev(cases[0][1])
        q_d, k_d, bt, cu = G.bf16_dev(q), G.cache_dev(kc), G.dev(b.block_table), G.dev(b.cu_seqlens_q)
        desc = ea.make_desc(b.geom, num_seqs=3, num_q_tokens=len(q), max_q_len=max(q_lens), max_kv_len=1200,
                            max_blocks_per_seq=bt.shape[1], num_blocks=k_d.shape[0])
        ws = torch.empty(max(1, ea.kv_score_workspace_bytes(desc)), dtype=torch.uint8, device="cuda")
        run = lambda: ea.kv_score(b.geom, q_d, lse_d, k_d, bt, lens_d, cu, w_d, max_q_len=max(q_lens),
                                  max_kv_len=1200, workspace=ws)
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        for turn in range(5):
            n, lse, ref = cases[turn % 3]
            lens_d.copy_(G.dev(n))
            lse_d.copy_(G.dev(lse))
            w_d.copy_(G.dev(w))
            ws.fill_(255)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = w_d.cpu().numpy()
            assert (np.abs(got - ref) <= REL * ref + 1e-7).all()
            w_d.copy_(G.dev(w))
            run()
            assert np.array_equal(got, w_d.cpu().numpy())


def test_selection_of_sequences_longer_than_announced(G):
    b = R.make_batch([9000, 40000, 300], [1] * 3, num_kv_heads=2)
    rng = np.random.default_rng(5)
    w = rng.random((b.num_blocks, 2, 16)).astype(np.float32)
    ref, ref_counts = R.kv_select(b, w, 700, 4, 64)
    for bound in (300, 8192, 9000, 40000):
        keep, counts = ea.kv_select(b.geom, G.dev(w), G.dev(b.block_table), G.dev(b.seq_lens), budget=700,
                                    keep_first=4, keep_last=64, max_kv_len=bound)
        assert np.array_equal(counts.cpu().numpy(), ref_counts) and np.array_equal(keep.cpu().numpy(), ref)


def test_tensors_that_do_not_fit_are_refused(G):
    b, q, kc, vc, ks, vs, sinks = R.filled([50, 30], [4, 1], num_kv_heads=2)
    g, lse = b.geom, np.zeros((5, 16), np.float32)
    w = torch.zeros((b.num_blocks, 2, 16), device="cuda")
    base = dict(q=G.bf16_dev(q), lse=G.dev(lse), k_cache=G.cache_dev(kc), block_table=G.dev(b.block_table),
                seq_lens=G.dev(b.seq_lens), cu_seqlens_q=G.dev(b.cu_seqlens_q), scores=w)
    def bad(f, good, *changes):
        for change in changes:
            with pytest.raises((ValueError, TypeError, ea.EidError)):
                f(g, **{**good, **change})
    hints = dict(max_q_len=4, max_kv_len=50)
    ea.kv_score(g, **base, **hints)
    bad(lambda *a, **k: ea.kv_score(*a, **{**hints, **k}), base,
        dict(q=base["q"].float()), dict(q=base["q"][:, :8]), dict(q=base["q"].cpu()), dict(q=base["q"][:4]),
        dict(lse=base["lse"].double()), dict(lse=base["lse"].t()), dict(k_cache=base["k_cache"][:, :8]),
        dict(scores=w[:-1]), dict(scores=w.half()), dict(seq_lens=base["seq_lens"].long()), dict(seq_lens=None),
        dict(cu_seqlens_q=base["cu_seqlens_q"][:2]), dict(max_kv_len=50000), dict(max_q_len=0))
    tree = dict(q=base["q"], k_cache=base["k_cache"], v_cache=G.cache_dev(vc), block_table=base["block_table"],
                seq_lens=base["seq_lens"], cu_seqlens_q=base["cu_seqlens_q"],
                tree_mask=torch.ones((5, 1), dtype=torch.int64, device="cuda"))
    ea.attn_tree(g, **tree, **hints)
    bad(lambda *a, **k: ea.attn_tree(*a, **{**hints, **k}), tree,
        dict(tree_mask=tree["tree_mask"].int()), dict(tree_mask=tree["tree_mask"][:4]), dict(v_cache=tree["v_cache"].cpu()),
        dict(v_cache=tree["v_cache"][:-1]), dict(max_q_len=300), dict(out=torch.empty_like(base["q"])[:, ::2]),
        dict(sinks=torch.zeros(3, device="cuda")), dict(max_kv_len=0),
        dict(workspace=torch.empty(0, dtype=torch.uint8)))
    sel = dict(scores=w, block_table=base["block_table"], seq_lens=base["seq_lens"])
    hints = dict(budget=20, max_kv_len=50)
    keep, counts = ea.kv_select(g, **sel, **hints)
    bad(lambda *a, **k: ea.kv_select(*a, **{**hints, **k}), sel,
        dict(scores=w[:, :1]), dict(scores=w.double()), dict(budget=0), dict(keep_first=15, keep_last=6),
        dict(keep=keep[:, :, :10]), dict(counts=counts.long()), dict(max_kv_len=10 ** 6), dict(block_table=None))
    k1, v1 = base["k_cache"], tree["v_cache"]
    com = dict(k_caches=[k1], v_caches=[v1], block_table=base["block_table"], seq_lens=base["seq_lens"], keep=keep,
               counts=counts)
    bad(ea.kv_compact, com, dict(v_caches=[k1]), dict(k_caches=[k1, k1], v_caches=[v1, v1]), dict(k_caches=[]),
        dict(k_caches=[k1, v1]), dict(scores=[w, w]), dict(scores=[w.half()]), dict(keep=keep.long()),
        dict(keep=keep[:1]), dict(counts=counts[:1]), dict(starts=counts.float()), dict(k_caches=[k1[:-1]]),
        dict(k_caches=[k1.transpose(1, 2)]))


@pytest.mark.parametrize("kv_dtype", [KV_BF16, KV_FP8_E4M3])
@pytest.mark.parametrize("heads", [4, 24])
def test_other_head_counts(G, heads, kv_dtype):
    for q_lens in ([1, 2, 1], [1, 40, 3]):
        b, q, kc, vc, ks, vs, sinks = R.filled([130, 70, 33], q_lens, num_kv_heads=heads, kv_dtype=kv_dtype)
        lse = lse_of(b, q, kc, vc, sinks, ks, vs)
        w = pool(b, np.random.default_rng(8))
        ref = R.kv_score(b, q, lse, kc, w, ks)
        assert (np.abs(score(G, b, q, lse, kc, w, ks) - ref) <= REL * ref + 1e-7).all()
    keep, counts = select(G, b, w, 30, 2, 5)
    ref, ref_counts = R.kv_select(b, w, 30, 2, 5)
    assert np.array_equal(keep, ref) and np.array_equal(counts, ref_counts)
    kd, vd, wd = G.cache_dev(kc), G.cache_dev(vc), G.dev(w)
    ea.kv_compact(b.geom, [kd], [vd], G.dev(b.block_table), G.dev(b.seq_lens), G.dev(keep), G.dev(counts), scores=[wd])
    assert np.array_equal(G.cache_host(kd), R.kv_compact(b, kc, keep, counts, [0] * 3, True))
    assert np.array_equal(G.cache_host(vd), R.kv_compact(b, vc, keep, counts, [0] * 3, True))
    # the same rows in every head, behind the context
    path = np.sort(np.random.default_rng(9).choice(np.arange(20, 33), (3, 6), replace=True), axis=1).astype(np.int32)
    path = np.maximum(path, 20 + np.arange(6, dtype=np.int32))
    starts, n = np.full(3, 20, np.int32), np.array([6, 0, 4], np.int32)
    kd = G.cache_dev(kc)
    ea.kv_compact(b.geom, [kd], [vd], G.dev(b.block_table), G.dev(b.seq_lens), G.dev(path), G.dev(n), starts=G.dev(starts))
    assert np.array_equal(G.cache_host(kd), R.kv_compact(b, kc, path, n, starts, False))


def test_pages_past_two_to_the_32_bytes(G):
    # scores, selections and moves in pages whose byte offsets in the cache do not fit 32 bits
    nb = (1 << 32) // 16384 + 40
    b, q, kc, vc, ks, vs, sinks = R.filled([100, 60], [1, 2])
    far = nb - kc.shape[0]
    k, v = (torch.zeros((nb, 16, 8, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    w = torch.zeros((nb, 8, 16), device="cuda")
    bt, sl, cu = G.dev((b.block_table + far).astype(np.int32)), G.dev(b.seq_lens), G.dev(b.cu_seqlens_q)
    for t, c in ((k, kc), (v, vc)):
        t[far:] = G.cache_dev(c)
    start = pool(b, np.random.default_rng(2))
    lse = lse_of(b, q, kc, vc, sinks, ks, vs)
    ref = R.kv_score(b, q, lse, kc, start)
    for max_q in (2, 3):                       # the kernels for few rows and for any number
        w[far:] = G.dev(start)
        ea.kv_score(b.geom, G.bf16_dev(q), G.dev(lse), k, bt, sl, cu, w, max_q_len=max_q, max_kv_len=100)
        assert (np.abs(w[far:].cpu().numpy() - ref) <= REL * ref + 1e-7).all()
    got = w[far:].cpu().numpy()
    keep, counts = ea.kv_select(b.geom, w, bt, sl, budget=40, keep_first=2, keep_last=3, max_kv_len=100)
    rk, rc = R.kv_select(b, got, 40, 2, 3)
    assert np.array_equal(keep.cpu().numpy(), rk) and np.array_equal(counts.cpu().numpy(), rc)
    ea.kv_compact(b.geom, [k], [v], bt, sl, keep, counts, scores=[w])
    assert np.array_equal(G.cache_host(k[far:].contiguous()), R.kv_compact(b, kc, rk, rc, [0, 0], True))
    assert np.array_equal(G.cache_host(v[far:].contiguous()), R.kv_compact(b, vc, rk, rc, [0, 0], True))
    assert not k[:far].any() and not w[:far].any()
