"""Refusals and planning of the tree attention and of the operators that thin a cache out, and the
scheduler's truncation: host code, no GPU."""
import ctypes as C

import numpy as np
import pytest

import eidola_amd as ea
from eidola_amd import _lib
from eidola_amd._lib import AttnArgs

import cache_ref as R

BAD, UNSUP, WS = _lib.EID_ERR_INVALID_ARG, _lib.EID_ERR_UNSUPPORTED, _lib.EID_ERR_WORKSPACE


def desc(geom=None, **kw):
    d = ea.make_desc(geom or ea.AttnGeometry(), num_seqs=4, num_q_tokens=40, max_q_len=16, max_kv_len=1000,
                     max_blocks_per_seq=63, num_blocks=128)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def args(d, **kw):
    a = AttnArgs()
    for f in ("q", "out", "k_cache", "v_cache", "block_table", "seq_lens", "cu_seqlens_q"):
        setattr(a, f, 0x1000)
    a.workspace, a.workspace_bytes = 0x2000, ea.attn_tree_workspace_bytes(d)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def tree(d, a, mask=0x3000, words=1):
    return ea.load_library().eid_attn_tree(C.byref(d), C.byref(a), mask, words, None)


@pytest.mark.parametrize("kw,status", [
    (dict(head_dim=128), UNSUP), (dict(num_q_heads=32), UNSUP), (dict(num_seqs=0), BAD), (dict(max_q_len=41), BAD),
    (dict(max_kv_len=5000), BAD), (dict(window=-1), BAD), (dict(softmax_scale=float("inf")), BAD),
    (dict(num_q_tokens=300, max_q_len=257), UNSUP), (dict(struct_size=8), BAD),
])
def test_tree_descriptors_refused(kw, status):
    d = desc(**kw)
    assert ea.attn_tree_workspace_bytes(d) == 0
    assert tree(d, args(d)) == status and ea.load_library().eid_last_error()


def test_tree_arguments_refused():
    d = desc()
    assert ea.attn_tree_workspace_bytes(d) > 0
    assert tree(d, args(d), mask=None) == BAD
    assert tree(d, args(d), mask=0x3004) == BAD
    assert tree(d, args(d), words=0) == BAD and tree(d, args(d), words=5) == BAD
    big = desc(num_q_tokens=100, max_q_len=65)
    assert tree(big, args(big), words=1) == BAD
    for f in ("q", "out", "k_cache", "v_cache", "block_table", "seq_lens", "cu_seqlens_q"):
        assert tree(d, args(d, **{f: None})) == BAD
    assert tree(d, args(d, q=0x1008)) == BAD
    assert tree(d, args(d, k_new=0x1000)) == BAD
    assert tree(d, args(d, workspace=None)) == WS
    assert tree(d, args(d, workspace=0x2010)) == WS
    assert tree(d, args(d, workspace_bytes=ea.attn_tree_workspace_bytes(d) - 1)) == WS
    assert tree(desc(kv_dtype=ea.KV_FP8_E4M3), args(d)) == BAD
    assert ea.load_library().eid_attn_tree(C.byref(d), None, 0x3000, 1, None) == BAD
    assert ea.load_library().eid_attn_tree(None, None, 0x3000, 1, None) == BAD


def test_tree_workspace_follows_the_bounds():
    small = ea.attn_tree_workspace_bytes(desc(max_kv_len=64, max_q_len=4))
    large = ea.attn_tree_workspace_bytes(desc())
    assert 0 < small <= large
    assert ea.attn_tree_workspace_bytes(desc(sum_kv_len=1000)) <= large
    assert ea.attn_tree_workspace_bytes(desc(window=16)) <= large
    # a bounded workspace, whatever the batch
    huge = desc(num_seqs=60000, num_q_tokens=60000 * 16, max_kv_len=1000)
    assert ea.attn_tree_workspace_bytes(huge) <= 256 << 20


def test_score_refusals():
    lib, ok = ea.load_library(), 0x1000
    call = lambda d, q=ok, lse=ok, k=ok, bt=ok, cu=ok, sl=ok, ks=None, w=ok, ws=None, n=0: lib.eid_kv_score(
        C.byref(d) if d else None, q, lse, k, bt, cu, sl, ks, w, ws, n, None)
    assert call(None) == BAD and call(desc(head_dim=32)) == UNSUP and call(desc(max_kv_len=0)) == BAD
    for f in ("q", "lse", "k", "bt", "cu", "sl", "w"):
        assert call(desc(), **{f: None}) == BAD
    for f in ("q", "lse", "k", "w"):
        assert call(desc(), **{f: 0x1004}) == BAD
    assert call(desc(kv_dtype=ea.KV_FP8_E4M3)) == BAD
    # a long chunk whose rows are shared out needs a workspace; few rows do not
    assert ea.kv_score_workspace_bytes(desc()) == 0 and ea.kv_score_workspace_bytes(desc(num_seqs=0)) == 0
    long = desc(num_seqs=1, num_q_tokens=512, max_q_len=512)
    need = ea.kv_score_workspace_bytes(long)
    assert need > 0 and call(long) == WS and call(long, ws=0x2000, n=need - 1) == WS
    assert call(long, ws=0x2010, n=need) == WS
    assert ea.kv_score_workspace_bytes(desc(num_seqs=512, num_q_tokens=512 * 512, max_q_len=512)) == 0


def test_select_refusals():
    lib, ok = ea.load_library(), 0x1000
    call = lambda d, w=ok, bt=ok, sl=ok, budget=64, first=4, last=16, keep=ok, counts=ok: lib.eid_kv_select(
        C.byref(d) if d else None, w, bt, sl, budget, first, last, keep, counts, None)
    assert call(None) == BAD and call(desc(num_seqs=0)) == BAD and call(desc(max_blocks_per_seq=0)) == BAD
    assert call(desc(num_seqs=70000)) == UNSUP and call(desc(max_blocks_per_seq=1 << 30)) == UNSUP
    assert call(desc(), budget=0) == BAD and call(desc(), budget=-3) == BAD
    assert call(desc(), first=-1) == BAD and call(desc(), last=-1) == BAD
    assert call(desc(), first=50, last=15) == BAD and call(desc(), first=2 ** 31 - 1, last=2 ** 31 - 1) == BAD
    for f in ("w", "bt", "sl", "keep", "counts"):
        assert call(desc(), **{f: None}) == BAD
    assert call(desc(), w=0x1004) == BAD


def test_compact_refusals():
    lib, ok = ea.load_library(), 0x1000
    two, hole, odd = (C.c_int64 * 2)(ok, ok), (C.c_int64 * 2)(ok, 0), (C.c_int64 * 2)(ok, ok + 8)

    def call(d, n=2, k=two, v=two, w=None, bt=ok, sl=ok, keep=ok, strides=(0, 8, 0), rows=8, counts=ok, starts=None):
        return lib.eid_kv_compact(C.byref(d) if d else None, n, k, v, w, bt, sl, keep, *strides, rows, counts, starts,
                                  None)
    assert call(None) == BAD and call(desc(block_size=8)) == UNSUP
    assert call(desc(), n=-1) == BAD and call(desc(), rows=-1) == BAD
    assert call(desc(), n=0) == 0 and call(desc(), rows=0) == 0       # nothing to move
    for f in ("k", "v", "bt", "sl", "keep", "counts"):
        assert call(desc(), **{f: None}) == BAD
    for f in ("k", "v", "w"):
        assert call(desc(), **{f: hole}) == BAD and call(desc(), **{f: odd}) == BAD
    for i in range(3):
        strides = [0, 8, 0]
        strides[i] = -8
        assert call(desc(), strides=strides) == BAD


def test_the_reference_of_the_gpu_tests_agrees_with_the_oracle():
    # a chain of drafted tokens is causal attention: the C oracle computes that too
    import oracle
    from helpers import desc_of
    for window in (0, 3):
        b, q, kc, vc, ks, vs, sinks = R.filled([30, 9], [5, 9], num_kv_heads=1, window=window)
        mask = R.tree_masks([list(range(-1, n - 1)) for n in (5, 9)], 1)
        out, lse = R.attn_tree(b, q, kc, vc, mask, sinks)
        ref, ref_lse = oracle.attn_f64(desc_of(b), q, kc, vc, b.block_table, b.seq_lens, b.cu_seqlens_q, sinks,
                                       None, None)
        assert np.allclose(out, ref, atol=1e-9) and np.allclose(lse, ref_lse, atol=1e-6)
    # masks of several words: bits land where they were put
    m = R.masks_from_ints([1 << 63 | 1, 1 << 64, 1 << 130 | 3], 3)
    bits = R.mask_bits(m, 140)
    assert [np.nonzero(r)[0].tolist() for r in bits] == [[0, 63], [64], [0, 1, 130]]
    import torch
    codes = torch.arange(256, dtype=torch.int32).to(torch.uint8)
    assert np.array_equal(R.fp8_f64(codes.numpy()), codes.view(torch.float8_e4m3fn).double().numpy(), equal_nan=True)


# ---- truncation --------------------------------------------------------------------------------

def test_truncate_gives_pages_back_and_appends_go_on():
    s = ea.Scheduler(num_blocks=8, max_blocks_per_seq=8)
    s.add_seq(1)
    b = s.build_batch([1], [70])                       # 5 blocks
    assert s.free_blocks == 3
    s.truncate(1, 33, 20)                              # 3 blocks stay
    assert s.seq_len(1) == 33 and s.free_blocks == 5
    d = s.build_batch([1], [2])
    assert d.positions.tolist() == [33, 34] and d.block_table[0, :3].tolist() == b.block_table[0, :3].tolist()
    assert d.slot_mapping.tolist() == [int(b.block_table[0, 2]) * 16 + 1, int(b.block_table[0, 2]) * 16 + 2]
    s.truncate(1, 35)                                  # nothing to cut
    s.truncate(1, 0)
    assert s.seq_len(1) == 0 and s.free_blocks == 8
    assert s.build_batch([1], [1]).positions.tolist() == [0]


@pytest.mark.parametrize("new_len,unchanged", [(-1, -1), (71, 71), (10, 11), (10, -1)])
def test_truncate_refusals(new_len, unchanged):
    s = ea.Scheduler(num_blocks=8, max_blocks_per_seq=8)
    s.add_seq(1)
    s.build_batch([1], [70])
    with pytest.raises(ea.EidError) as e:
        s.truncate(1, new_len, unchanged)
    assert e.value.name == "EID_ERR_INVALID_ARG" and s.seq_len(1) == 70 and s.free_blocks == 3
    with pytest.raises(ea.EidError):
        s.truncate(2, 0)
    assert ea.load_library().eid_sched_truncate(None, 1, 0, 0) == BAD


def tokens(n, seed=0):
    return np.random.default_rng(seed).integers(0, 1000, n).astype(np.int32)


def test_truncated_prefix_is_still_matched_and_goes_on():
    t = tokens(64)
    s = ea.Scheduler(num_blocks=16, max_blocks_per_seq=8, prefix_reuse=True)
    s.add_seq(1, t)
    s.build_batch([1], [64], t)
    s.truncate(1, 40)                                  # blocks 0, 1 whole, 8 rows in block 2
    assert s.add_seq(2, t) == 32                       # block 2 is open again: no longer matched
    # the chain goes on from row 40: the same tokens lead to the same blocks' hashes
    s.build_batch([1], [24], t[40:])
    assert s.add_seq(3, np.concatenate([t, t[:1]])) == 64
    # within a partly filled block
    u = tokens(30, 1)
    s.add_seq(4, u)
    s.build_batch([4], [30], u)
    s.truncate(4, 20)
    s.build_batch([4], [13], np.concatenate([u[20:], u[:3]]))
    assert s.add_seq(5, np.concatenate([u, u[:4]])) == 32


def test_rewritten_rows_leave_the_index():
    t = tokens(80)
    s = ea.Scheduler(num_blocks=32, max_blocks_per_seq=8, prefix_reuse=True)
    s.add_seq(1, t)
    s.build_batch([1], [80], t)
    s.truncate(1, 48, 16)                              # rows 16 .. 47 hold others now
    assert s.add_seq(2, t) == 16
    s.build_batch([1], [32], tokens(32, 2))            # later blocks are not indexed either
    assert s.add_seq(3, np.concatenate([t[:48], tokens(32, 2), t[:1]])) == 16


def test_shared_blocks_may_not_be_rewritten_or_opened():
    t = tokens(64)
    s = ea.Scheduler(num_blocks=16, max_blocks_per_seq=8, prefix_reuse=True)
    s.add_seq(1, t)
    s.build_batch([1], [64], t)
    assert s.add_seq(2, np.concatenate([t, t])) == 64
    free = s.free_blocks
    for new_len, unchanged in ((60, 60), (64, 48), (32, 0), (64, 63)):
        with pytest.raises(ea.EidError):
            s.truncate(2, new_len, unchanged)
        assert s.seq_len(2) == 64 and s.free_blocks == free
    s.truncate(2, 48)                                  # whole blocks may be given back
    assert s.seq_len(2) == 48 and s.free_blocks == free and s.add_seq(3, np.concatenate([t, t])) == 64


def test_random_truncations_keep_the_books():
    rng = np.random.default_rng(5)
    s = ea.Scheduler(num_blocks=64, max_blocks_per_seq=16, prefix_reuse=True)
    have = {}
    for turn in range(400):
        act = rng.integers(0, 4)
        if act == 0 and len(have) < 6:
            sid = turn
            p = tokens(int(rng.integers(1, 60)), int(rng.integers(0, 3)))
            have[sid] = (list(p), s.add_seq(sid, p))
        elif have:
            sid = int(rng.choice(list(have)))
            toks, n = have[sid]
            if act == 1:
                k = int(rng.integers(1, 20))
                new = (list(toks[n:n + k]) + list(tokens(k, turn)))[:k]
                if n + k <= 256:
                    try:
                        s.build_batch([sid], [k], np.array(new, np.int32))
                        have[sid] = (toks[:n] + new, n + k)
                    except ea.EidError as e:
                        assert e.name == "EID_ERR_NO_BLOCKS"
            elif act == 2:
                cut = int(rng.integers(0, n + 1))
                try:
                    s.truncate(sid, cut)
                    have[sid] = (toks[:cut], cut)
                except ea.EidError as e:
                    assert e.name == "EID_ERR_INVALID_ARG"
            else:
                s.free_seq(sid)
                del have[sid]
        for sid, (toks, n) in have.items():
            assert s.seq_len(sid) == n
        refs = [s.block_refs(i) for i in range(64)]
        assert refs.count(0) == s.free_blocks
        assert sum(refs) == sum((n + 15) // 16 for _, n in have.values())
