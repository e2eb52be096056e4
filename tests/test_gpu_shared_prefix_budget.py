"""Caches cut to a budget, and drafted trees committed, while the scheduler shares prefixes: the new length first, which
is refused where pages are shared, then the move.  Rows are compared bit for bit."""
import numpy as np
import pytest
import torch

import eidola_amd as ea

import cache_ref as R

pytestmark = pytest.mark.gpu
GEOM = ea.AttnGeometry(num_q_heads=16, num_kv_heads=2)
BLOCKS, BUDGET = 48, 96


def d(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Pool:
    """A scheduler with two layers of caches and scores, whose rows are all different."""

    def __init__(self):
        self.sched = ea.Scheduler(BLOCKS, BLOCKS, prefix_reuse=True)
        rows = torch.arange(BLOCKS * 16 * 2, device="cuda").view(BLOCKS, 16, 2, 1)
        self.kc, self.vc = ([((rows * 7 + 13 * i + torch.arange(64, device="cuda")) % 251).to(torch.bfloat16)
                             for i in range(2)] for _ in range(2))
        for v in self.vc:
            v.neg_()
        g = torch.Generator(device="cuda").manual_seed(1)
        self.scores = [torch.rand((BLOCKS, 2, 16), device="cuda", generator=g) for _ in range(2)]

    def add(self, seq, tokens):
        """The sequence with all its tokens; how many of them the index had."""
        tokens = np.asarray(tokens, np.int32)
        had = self.sched.add_seq(seq, tokens)
        self.batch = self.sched.build_batch([seq], [len(tokens) - had], tokens[had:])
        return had

    def rows(self, batch, layer, n):
        """The first n rows of every tensor of a layer, as the batch's block table has them."""
        at = d(batch.block_table[0].astype(np.int64))[torch.arange(n, device="cuda") // 16]
        j = torch.arange(n, device="cuda") % 16
        return [self.kc[layer][at, j], self.vc[layer][at, j], self.scores[layer][at, :, j]]

    def cut(self, seq, batch, first, last=16):
        """A sequence to its budget, in both layers."""
        n = int(batch.seq_lens[0])
        self.sched.truncate(seq, BUDGET, first)
        bt, sl = d(batch.block_table), d(batch.seq_lens)
        keeps = [ea.kv_select(GEOM, w, bt, sl, budget=BUDGET, keep_first=first, keep_last=last, max_kv_len=n)
                 for w in self.scores]
        keep = torch.stack([k for k, _ in keeps])
        ea.kv_compact(GEOM, self.kc, self.vc, bt, sl, keep, keeps[0][1], scores=self.scores)
        return keep.cpu().numpy()


def tokens(n, seed):
    return np.random.default_rng(seed).integers(0, 1000, n).astype(np.int32)


def test_a_shared_prefix_survives_its_other_owners_budget():
    p = Pool()
    t = tokens(160, 0)
    assert p.add(1, t[:80]) == 0
    one = p.batch
    assert p.add(2, t) == 80
    two = p.batch
    first = [x.clone() for l in range(2) for x in p.rows(one, l, 80)]
    second = [p.rows(two, l, 160) for l in range(2)]
    everything = [x.clone() for x in p.kc + p.vc + p.scores]
    # rows of the shared pages would change: refused, and nothing is moved
    free = p.sched.free_blocks
    with pytest.raises(ea.EidError) as e:
        p.cut(2, two, first=4)
    assert e.value.name == "EID_ERR_INVALID_ARG"
    assert p.sched.seq_len(2) == 160 and p.sched.free_blocks == free
    assert all(torch.equal(a, b) for a, b in zip(everything, p.kc + p.vc + p.scores))
    # with the shared rows kept where they are the cut leaves them to their other owner
    keep = p.cut(2, two, first=80)
    assert p.sched.seq_len(2) == BUDGET and p.sched.free_blocks == free + 4
    assert all(torch.equal(a, b) for a, b in zip(first, [x for l in range(2) for x in p.rows(one, l, 80)]))
    for l in range(2):
        for old, new in zip(second[l], p.rows(two, l, BUDGET)):
            for h in range(2):
                assert torch.equal(new[:, h], old[d(keep[l, 0, h].astype(np.int64)), h])
    # the prefix is still matched, what was rewritten is not
    assert p.sched.add_seq(3, t) == 80


def test_pages_given_back_before_the_move_may_be_written_behind_it():
    p = Pool()
    t = tokens(300, 1)
    p.add(1, t)
    batch = p.batch
    before = [p.rows(batch, l, 300) for l in range(2)]
    keep = p.cut(1, batch, first=4)
    # another sequence takes every free page, those that the move has read among them, and writes its rows
    q_len = p.sched.free_blocks * 16
    p.sched.add_seq(2)
    other = p.sched.build_batch([2], [q_len], tokens(q_len, 2))
    assert set(other.block_table[0, :q_len // 16]) & set(batch.block_table[0, :19])
    k = torch.full((q_len, 2, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    for l in range(2):
        ea.kv_write(GEOM, k, k, p.kc[l], p.vc[l], d(other.slot_mapping))
    for l in range(2):
        for old, new in zip(before[l], p.rows(batch, l, BUDGET)):
            for h in range(2):
                assert torch.equal(new[:, h], old[d(keep[l, 0, h].astype(np.int64)), h])
    assert p.sched.add_seq(3, t) == 0                  # (block 0 holds row 4 and up, which changed)


def test_an_accepted_path_behind_a_shared_prefix():
    p = Pool()
    t = tokens(65, 3)
    assert p.add(1, t[:64]) == 0
    one = p.batch
    assert p.add(2, t) == 64
    tree = p.sched.build_batch([2], [6])               # rows 65 .. 70, without tokens
    first = [x.clone() for l in range(2) for x in p.rows(one, l, 64)]
    old = [p.rows(tree, l, 71) for l in range(2)]
    path = [0, 2, 5]
    p.sched.truncate(2, 68, 65)
    ea.kv_compact(GEOM, p.kc, p.vc, d(tree.block_table), d(tree.seq_lens),
                  d(np.array([[65 + i for i in path]], np.int32)), d(np.array([3], np.int32)),
                  starts=d(np.array([65], np.int32)))
    assert p.sched.seq_len(2) == 68
    assert all(torch.equal(a, b) for a, b in zip(first, [x for l in range(2) for x in p.rows(one, l, 64)]))
    for l in range(2):
        for a, b in zip(old[l][:2], p.rows(tree, l, 68)[:2]):
            assert torch.equal(b[:65], a[:65]) and torch.equal(b[65:], a[[65 + i for i in path]])
