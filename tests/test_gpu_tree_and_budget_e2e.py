"""The operators as an engine strings them together, over the scheduler's own pages.

Drafted trees: a two-layer attention stack (a windowed and a full layer, random weights) decodes
greedily; beside it another sequence of the same prompt verifies drafted trees, keeps the accepted path
(kv_compact over both layers, Scheduler.truncate) and goes on.  Logits of accepted tokens must be those of the
plain decode: both run the same kernels' arithmetic on the same tokens, apart from the order of
sums and bf16 roundings in between.

Budget: a sequence's cache is cut while it decodes; attention over what is left must equal the
64-bit attention over exactly the rows that a plain restatement keeps."""
import numpy as np
import pytest
import torch

import eidola_amd as ea

import cache_ref as R
from helpers import MAX_ABS_TOL

pytestmark = pytest.mark.gpu
H, VOCAB = 512, 320


class Stack:
    """Layers with windows (8, 0) over one scheduler; hidden size 512, 16 query heads on 2 KV heads."""

    def __init__(self, seed, windows=(8, 0), blocks=64):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s, k: (torch.randn(s, device="cuda", generator=g) * k).to(torch.bfloat16)
        self.geoms = [ea.AttnGeometry(num_q_heads=16, num_kv_heads=2, window=w) for w in windows]
        self.emb = r(VOCAB, H, k=1.0)
        self.wqkv = [r(20 * 64, H, k=0.06) for _ in windows]
        self.wo = [r(H, 16 * 64, k=0.05) for _ in windows]
        self.sinks = [torch.randn(16, device="cuda", generator=g) for _ in windows]
        self.kc = [torch.full((blocks, 16, 2, 64), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in windows]
        self.vc = [torch.full_like(k, float("nan")) for k in self.kc]
        self.cos_sin = torch.from_numpy(ea.yarn_cos_sin(1024)).cuda()
        self.sched = ea.Scheduler(blocks, 16)

    def step(self, seq, tokens, positions=None, mask=None):
        """Appends the tokens to the sequence; logits of every one of them."""
        n = len(tokens)
        b = self.sched.build_batch([seq], [n])
        d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
        bt, sl, cu, slots = d(b.block_table), d(b.seq_lens), d(b.cu_seqlens_q), d(b.slot_mapping)
        pos = d(b.positions if positions is None else np.asarray(positions, np.int32))
        x = self.emb[torch.tensor(tokens, device="cuda")].clone()
        norm = lambda h: (h.float() * torch.rsqrt(h.float().pow(2).mean(-1, keepdim=True) + 1e-6)).to(torch.bfloat16)
        for l, g in enumerate(self.geoms):
            q = ea.rope_kv_write(g, ea.o_proj(norm(x), self.wqkv[l]), pos, self.cos_sin, self.kc[l], self.vc[l], slots)
            kw = dict(max_q_len=n, max_kv_len=b.max_kv_len, sinks=self.sinks[l])
            if mask is None:
                a = ea.attn_varlen(g, q, self.kc[l], self.vc[l], bt, sl, cu, **kw)
            else:
                a = ea.attn_tree(g, q, self.kc[l], self.vc[l], bt, sl, cu, d(mask), **kw)
            ea.o_proj(a, self.wo[l], residual=x, out=x)
        return (norm(x).float() @ self.emb.float().t()) / H ** 0.5, bt, sl

    def commit(self, bt, sl, seq, prefix, path):
        """Keeps the rows prefix + path[i] of a verified tree."""
        d = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
        ea.kv_compact(self.geoms[0], self.kc, self.vc, bt, sl, d([[prefix + i for i in path]]), d([len(path)]),
                      starts=d([prefix]))
        self.sched.truncate(seq, prefix + len(path), prefix)


def test_verified_trees_reproduce_the_plain_decode():
    m = Stack(3)
    rng = np.random.default_rng(0)
    prompt = rng.integers(0, VOCAB, 37).tolist()
    m.sched.add_seq(1)
    m.sched.add_seq(2)
    # plain decode: sequence 1
    logits = [m.step(1, prompt)[0][-1]]
    truth = [int(logits[-1].argmax())]
    for _ in range(40):
        lg, _, _ = m.step(1, [truth[-1]])
        logits.append(lg[-1])
        truth.append(int(lg[-1].argmax()))
    # drafted trees: sequence 2.  Token 0 is the last accepted token; the true continuation runs
    # through randomly placed nodes, the others are wrong drafts.
    lg, _, _ = m.step(2, prompt)
    done = 0                                            # truth[done] is the token to feed
    assert torch.allclose(lg[-1], logits[0], atol=0.05)
    while done < 34:
        n = int(rng.integers(2, 12))
        parents, toks, good = [-1], [truth[done]], [0]  # good: nodes on the true path
        for i in range(1, n):
            if len(good) < 5 and rng.random() < 0.5:
                parents.append(good[-1])
                toks.append(truth[done + len(good)])
                good.append(i)
            else:
                up = int(rng.integers(0, i))
                parents.append(up)
                toks.append((truth[done + 1] + 1 + int(rng.integers(0, VOCAB - 2))) % VOCAB)
        depth = []
        for p in parents:
            depth.append(0 if p < 0 else depth[p] + 1)
        prefix = m.sched.seq_len(2)
        lg, bt, sl = m.step(2, toks, [prefix + x for x in depth], R.tree_masks([parents], 1))
        for k, node in enumerate(good):
            assert torch.allclose(lg[node], logits[done + 1 + k], atol=0.05), (done, k)
        m.commit(bt, sl, 2, prefix, good)
        done += len(good)
        assert m.sched.seq_len(2) == len(prompt) + done
    # the first layer's rows depend on tokens and positions alone: bit for bit those of the decode
    rows = len(prompt) + done
    b = m.sched.build_batch([1, 2], [1, 1])
    at = [torch.from_numpy(b.block_table[s].astype(np.int64)).cuda() for s in (0, 1)]
    for cache in (m.kc[0], m.vc[0]):
        one, two = (cache[t].reshape(-1, 2, 64)[:rows].view(torch.int16) for t in at)
        assert torch.equal(one, two)


def test_a_cache_cut_to_its_budget_decodes_on():
    g = ea.AttnGeometry(num_q_heads=16, num_kv_heads=2)
    rng = np.random.default_rng(4)
    blocks, budget, first, last = 64, 96, 4, 16
    sched = ea.Scheduler(blocks, 32)
    sched.add_seq(5)
    sched.add_seq(6)
    kc = torch.full((blocks, 16, 2, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    vc = torch.full_like(kc, float("nan"))
    scores = torch.full((blocks, 2, 16), float("nan"), device="cuda")
    sinks = torch.from_numpy(rng.standard_normal(16).astype(np.float32)).cuda()
    # what should be in the cache: rows (K, V, score) per sequence and head, in 64 bits
    held = {s: [[] for _ in range(2)] for s in (5, 6)}

    def step(q_lens):
        ids = [5, 6]
        b = sched.build_batch(ids, q_lens)
        d = lambda a: torch.from_numpy(a).cuda()
        T = sum(q_lens)
        new = [torch.from_numpy(rng.standard_normal((T, h, 64)).astype(np.float32) * a).to(torch.bfloat16)
               for h, a in ((16, 2.0), (2, 1.0), (2, 1.0))]
        q, k, v = (t.cuda() for t in new)
        bt, sl, cu = d(b.block_table), d(b.seq_lens), d(b.cu_seqlens_q)
        ea.kv_write(g, k, v, kc, vc, d(b.slot_mapping))
        out, lse = ea.attn_varlen(g, q, kc, vc, bt, sl, cu, max_q_len=b.max_q_len, max_kv_len=b.max_kv_len,
                                  sinks=sinks, return_lse=True)
        ea.kv_score(g, q, lse, kc, bt, sl, cu, scores, max_q_len=b.max_q_len, max_kv_len=b.max_kv_len)
        qd, kd, vd = (t.double().numpy() for t in new)
        got = out.double().cpu().numpy()
        for i, s in enumerate(ids):
            a, e = b.cu_seqlens_q[i], b.cu_seqlens_q[i + 1]
            for h in range(2):
                rows = held[s][h]
                n_old = len(rows)
                rows += [[kd[r, h], vd[r, h], 0.0] for r in range(a, e)]
                K, V = np.stack([r[0] for r in rows]), np.stack([r[1] for r in rows])
                see = np.arange(len(rows))[None, :] <= n_old + np.arange(e - a)[:, None]
                ref, l = R.attn_rows(qd[a:e, 8 * h:8 * h + 8], K[:, None], V[:, None], see, 0.125,
                                     sinks[8 * h:8 * h + 8].cpu().numpy())
                assert np.abs(got[a:e, 8 * h:8 * h + 8] - ref).max() <= MAX_ABS_TOL
                for r in range(e - a):
                    p = np.exp(np.einsum("jd,xd->xj", K, qd[a + r, 8 * h:8 * h + 8]) * 0.125 - l[r][:, None])
                    for j in np.nonzero(see[r])[0]:
                        rows[j][2] += p[:, j].sum()
        return bt, sl, b

    cuts = 0
    bt, sl, b = step([150, 60])
    for turn in range(12):
        if max(b.seq_lens) > budget + 20 or turn == 0:
            cuts += 1
            keep, counts = ea.kv_select(g, scores, bt, sl, budget=budget, keep_first=first, keep_last=last,
                                        max_kv_len=b.max_kv_len)
            ea.kv_compact(g, [kc], [vc], bt, sl, keep, counts, scores=[scores])
            keep_h, counts_h = keep.cpu().numpy(), counts.cpu().numpy()
            for i, s in enumerate((5, 6)):
                n, L = int(counts_h[i]), int(b.seq_lens[i])
                assert n == min(L, budget)
                for h in range(2):
                    k = keep_h[i, h, :n]
                    assert (np.diff(k) > 0).all() and (keep_h[i, h, n:] == -1).all()
                    if L > budget:       # the rows that stay have the highest sums (fp32 apart)
                        w = np.array([r[2] for r in held[s][h]])
                        assert set(range(first)) <= set(k.tolist()) and set(range(L - last, L)) <= set(k.tolist())
                        mid = np.arange(first, L - last)
                        inside = np.isin(mid, k)
                        assert w[mid[inside]].min() >= w[mid[~inside]].max() * (1 - 1e-3)
                    held[s][h] = [held[s][h][j] for j in k]
                sched.truncate(s, n, min(n, first))
            assert sched.seq_len(5) == budget
        bt, sl, b = step([1 + 3 * (turn % 2), 1])
    assert cuts >= 2
