"""Cases of the cache operators beside the attention calls: attention for a tree of drafted
tokens, the attention weight every cached key has received, the choice of the rows that stay,
and the move that brings kept rows together.  Geometry of the package: 8 query heads per KV
head, head_dim 64, pages of 16 tokens, a bf16 or fp8-e4m3fn cache.

Where `own` is false run() computes the operators in elementary torch operations over padded
batches; where it is true it makes the package's calls."""
import math
import random

import torch

own = False

PAGE, GROUP, DIM = 16, 8, 64
SCALE = 0.125


def listed():
    tree = dict(op="tree", kv_heads=8, window=0, fp8=False, sinks=True, lse=False)
    score = dict(op="score", kv_heads=8, window=0, fp8=False)
    select = dict(op="select", kv_heads=8)
    return [
        # one user, a short chat, a handful of drafted tokens: what counts is the latency
        dict(tree, name="tree 1x8 @500", seqs=1, nodes=8, context=500, ragged=False),
        # a serving batch with small trees: the caches are read once, for a few rows
        dict(tree, name="tree 16x16 @8k ragged", seqs=16, nodes=16, context=8192, ragged=True, lse=True),
        # the same step on a layer with a sliding window: little to read, many sequences
        dict(tree, name="tree 32x24 @4k window", seqs=32, nodes=24, context=4096, ragged=True, window=128),
        # few users with long documents and wide trees: products, not bytes, are the bound
        dict(tree, name="tree 4x64 @32k", seqs=4, nodes=64, context=32768, ragged=False),
        # the same kind of step over a cache in 8 bits
        dict(tree, name="tree 8x32 @16k fp8", seqs=8, nodes=32, context=16384, ragged=True, fp8=True),
        # every decode step of a batch adds its attention weights
        dict(score, name="score 64x1 @8k", seqs=64, rows=1, context=8192, ragged=True),
        # a prompt chunk's rows add theirs: products over the whole context
        dict(score, name="score 1x2048 @4k", seqs=1, rows=2048, context=4096, ragged=False),
        # a mixed step over a cache in 8 bits: odd chunks next to single rows
        dict(score, name="score 8x37 @8k fp8", seqs=8, rows=37, context=8192, ragged=True, fp8=True),
        # one sequence has reached its budget
        dict(select, name="select 1 @3000", seqs=1, context=3000, budget=1000, ragged=False),
        # a batch of long ones is cut down together
        dict(select, name="select 32 @32k", seqs=32, context=32768, budget=4096, ragged=True),
        # accepted paths of a batch's trees, moved in the caches of all 36 layers
        dict(op="commit", name="commit 36 layers 16x32", kv_heads=8, layers=36, seqs=16, nodes=32, context=480,
             fp8=False, ragged=True),
        # a quarter of every sequence's rows stays, other rows in each KV head
        dict(op="compact", name="compact 8 @16k to 4k", kv_heads=8, seqs=8, context=16384, budget=4096, fp8=False,
             ragged=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "score", "score", "select", "commit", "compact"])
    heads = rng.choice([8, 8, 8, 2, 1])
    fp8 = rng.random() < 0.3
    ragged = rng.random() < 0.7
    seqs = _log(rng, 1, 64)
    if op == "tree":
        nodes = _log(rng, 1, 100)
        context = _log(rng, nodes + 1, max(nodes + 2, min(32768, 8_000_000 // (seqs * max(nodes, 45)))))
        return dict(op=op, seqs=seqs, nodes=nodes, context=context, kv_heads=heads, fp8=fp8, ragged=ragged,
                    window=rng.choice([0, 0, 128, rng.randint(1, 300)]), sinks=rng.random() < 0.7,
                    lse=rng.random() < 0.5)
    if op == "score":
        rows = rng.choice([1, _log(rng, 1, 40), _log(rng, 40, 1500)])
        context = _log(rng, rows, max(rows + 1, min(16384, 8_000_000 // (seqs * max(rows, 22)))))
        return dict(op=op, seqs=seqs, rows=rows, context=context, kv_heads=heads, fp8=fp8, ragged=ragged,
                    window=rng.choice([0, 0, 128]))
    context = _log(rng, 40, min(32768, 1_000_000 // seqs))
    if op == "select":
        return dict(op=op, seqs=seqs, context=context, budget=rng.randint(24, context + 20), kv_heads=heads,
                    ragged=ragged)
    if op == "commit":
        layers = rng.randint(1, 40)
        return dict(op=op, layers=layers, seqs=min(seqs, 16), nodes=_log(rng, 1, 64), context=_log(rng, 100, 480),
                    kv_heads=heads, fp8=fp8, ragged=ragged)
    context = min(context, 131072 // seqs)
    return dict(op=op, seqs=seqs, context=context, budget=rng.randint(24, context), kv_heads=heads, fp8=fp8,
                ragged=ragged)


def _lengths(case):
    """Cached tokens of every sequence (after this step's append) and its query rows."""
    n, top = case["seqs"], case["context"]
    rows = case.get("nodes", case.get("rows", 0))
    if not case["ragged"]:
        return [top] * n, [rows] * n
    q = [max(1, rows - (7 * s) % (rows // 2 + 1)) if rows else 0 for s in range(n)]
    if case["op"] == "score" and rows > 1:  # decode rows beside the chunks
        q = [1 if s % 3 == 2 else r for s, r in enumerate(q)]
    kv = [max(q[s], 1, int(top * (1 - 0.6 * ((s * 0.618) % 1.0)))) for s in range(n)]
    return kv, q


def work(case):
    kv, q = _lengths(case)
    h, elt = case["kv_heads"], 1 if case.get("fp8") else 2
    row = h * DIM * elt  # one token's keys (or values) in the cache
    op = case["op"]
    if op in ("tree", "score"):
        w = case["window"]
        keys = [min(k, w + n) if w else k for k, n in zip(kv, q)]
        if op == "tree":
            pairs = sum((min(w, k) if w else k) * n for k, n in zip(kv, q)) * h * GROUP
            return {"bytes": 2 * row * sum(keys) + 2 * 2 * sum(q) * h * GROUP * DIM, "flops": 4 * DIM * pairs}
        # a row sees the keys up to its own position
        pairs = sum(sum(min(w, k - n + i + 1) if w else k - n + i + 1 for i in range(n)) for k, n in zip(kv, q))
        return {"bytes": row * sum(keys) + 8 * h * sum(keys) + (2 * DIM + 4) * sum(q) * h * GROUP,
                "flops": 2 * DIM * pairs * h * GROUP}
    if op == "select":
        return {"bytes": 4 * h * (sum(kv) + len(kv) * case["budget"]), "flops": 0}
    if op == "commit":
        moved = sum(len(p) - 1 for p in _paths(case, 0))  # (the root stays where it is)
        return {"bytes": 2 * 2 * row * case["layers"] * max(1, moved), "flops": 0}
    kept = sum(min(k, case["budget"]) for k in kv)
    return {"bytes": 2 * (2 * row + 4 * h) * kept + 4 * h * kept, "flops": 0}


def _parents(case, s, seed):
    """Parent of every drafted token of sequence s; token 0 is the root."""
    r = random.Random(seed * 1009 + s)
    return [-1] + [r.randint(max(0, i - 9), i - 1) for i in range(1, _lengths(case)[1][s])]


def _paths(case, seed):
    """The accepted path of every sequence: node indices from the root on."""
    found = []
    for s in range(case["seqs"]):
        up, i, path = _parents(case, s, seed), 0, []
        i = len(up) - 1
        while i >= 0:
            path.append(i)
            i = up[i]
        found.append(path[::-1])
    return found


def _tree_bits(case, seed, words):
    """[rows, words] int64: bit j of a row says that the row's token descends from token j."""
    table = []
    for s in range(case["seqs"]):
        seen = []
        for i, up in enumerate(_parents(case, s, seed)):
            seen.append((seen[up] if up >= 0 else 0) | 1 << i)
        table += seen
    out = [[(m >> 64 * w) & (1 << 64) - 1 for w in range(words)] for m in table]
    return torch.tensor([[v - (1 << 64) if v >> 63 else v for v in m] for m in out], dtype=torch.int64)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv, q = _lengths(case)
    n, h, op = case["seqs"], case["kv_heads"], case["op"]
    pages = [(k + PAGE - 1) // PAGE for k in kv]
    total = sum(pages) + 3
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed))[: sum(pages)].to(torch.int32)
    table = torch.zeros((n, max(pages)), dtype=torch.int32)
    at = 0
    for s, m in enumerate(pages):
        table[s, :m] = order[at:at + m]
        at += m
    st = {"case": case, "kv": kv, "q_lens": q, "table": table.cuda(), "pages": total, "max_kv": max(kv), "sum_kv": sum(kv),
          "seq_lens": torch.tensor(kv, dtype=torch.int32).cuda()}

    def cache(layers=1):
        shape = (layers, total, PAGE, h, DIM)
        t = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        t.normal_(generator=g)
        if case["fp8"]:
            t = (t * 64).to(torch.float8_e4m3fn)  # (the scale beside it is 1/64)
        return t if layers > 1 or op == "commit" else t[0]

    st["keep_first"], st["keep_last"] = 4, 16
    if op in ("tree", "score"):
        rows = sum(q)
        st["k"] = cache()
        st["q"] = torch.randn((rows, h * GROUP, DIM), device="cuda", generator=g).to(torch.bfloat16)
        st["cu"] = torch.tensor([sum(q[:s]) for s in range(n + 1)], dtype=torch.int32).cuda()
        if case["fp8"]:  # keys' scales differ by head, as amax scales do
            st["ks"] = (torch.rand(h, device="cuda", generator=g) + 0.5) / 64
            st["vs"] = (torch.rand(h, device="cuda", generator=g) + 0.5) / 64
    if op == "tree":
        st["v"] = cache()
        st["mask"] = _tree_bits(case, seed, (max(q) + 63) // 64).cuda()
        st["sinks"] = torch.randn(h * GROUP, device="cuda", generator=g) if case["sinks"] else None
    elif op == "score":
        st["scores"] = torch.rand((total, h, PAGE), device="cuda", generator=g)
        s = _scores(st)[0]  # lse: what the attention call of this step has returned
        lse = torch.logsumexp(s, -1)
        del s
        st["lse"] = _rows(st, lse.view(n, h, max(q), GROUP).permute(0, 2, 1, 3).reshape(n, max(q), h * GROUP)).contiguous()
    elif op == "select":
        # few keys hold most of the weight; many have none to speak of, and some exactly none
        w = torch.rand((total, h, PAGE), device="cuda", generator=g)
        st["scores"] = w.pow(8) * 20 * (w > 0.2)
    else:
        st["k"], st["v"] = (cache(case["layers"]), cache(case["layers"])) if op == "commit" else (cache(), cache())
        if op == "commit":
            paths = _paths(case, seed)
            starts = [k - m for k, m in zip(kv, q)]
            most = max(map(len, paths))
            st["keep"] = torch.tensor([[b + i for i in p] + [-1] * (most - len(p)) for b, p in zip(starts, paths)],
                                      dtype=torch.int32).cuda()
            st["starts"] = torch.tensor(starts, dtype=torch.int32).cuda()
            st["counts"] = torch.tensor([len(p) for p in paths], dtype=torch.int32).cuda()
            st["layers_k"], st["layers_v"] = list(st["k"]), list(st["v"])
        else:
            st["scores"] = torch.rand((total, h, PAGE), device="cuda", generator=g)
            budget = case["budget"]
            rank = torch.rand((n, h, max(kv)), device="cuda", generator=g)
            j = torch.arange(max(kv), device="cuda")
            left = st["seq_lens"].view(n, 1, 1)
            rank = torch.where(j < left, rank, torch.full_like(rank, 2.0))
            first = rank.argsort(-1)[..., :budget]
            first = torch.where(first < left, first, torch.full_like(first, 1 << 30)).sort(-1).values
            keep = torch.full((n, h, budget), -1, dtype=torch.int32, device="cuda")
            keep[..., : first.shape[-1]] = torch.where(first < left, first, torch.full_like(first, -1)).to(torch.int32)
            st["keep"] = keep
            st["counts"] = torch.clamp(st["seq_lens"], max=budget)
    return st


# ---- the plain forms ------------------------------------------------------------------------

def _slots(st):
    """[sequences, longest] slot of every cached token (that of the last token behind the end)."""
    j = torch.arange(st["max_kv"], device="cuda")
    j = torch.minimum(j, st["seq_lens"].view(-1, 1).long() - 1)
    return torch.gather(st["table"].long(), 1, j // PAGE) * PAGE + j % PAGE


def _padded(st):
    """[sequences, longest] index of every query row, and which of them exist."""
    i = torch.arange(max(st["q_lens"]), device="cuda")
    cu = st["cu"].long()
    return torch.minimum(cu[:-1].view(-1, 1) + i, cu[1:].view(-1, 1) - 1), i < (cu[1:] - cu[:-1]).view(-1, 1)


def _of_pairs(lengths, lens_dev):
    """For every (sequence, place) below the lengths: its sequence and its place."""
    total = sum(lengths)
    lens = lens_dev.long()
    s = torch.repeat_interleave(torch.arange(len(lengths), device="cuda"), lens, output_size=total)
    return s, torch.arange(total, device="cuda") - (lens.cumsum(0) - lens)[s]


def _rows(st, x):
    """Rows [sequences, longest, ...] of a padded batch, one after the other."""
    s, i = _of_pairs(st["q_lens"], st["cu"][1:] - st["cu"][:-1])
    return x[s, i]


def _gathered(st, cache, scale):
    """[sequences, kv heads, tokens, dim] of a cache, in 32 bits."""
    h = st["case"]["kv_heads"]
    x = cache.reshape(-1, h, DIM)
    x = x.view(torch.uint8)[_slots(st)].view(torch.float8_e4m3fn) if st["case"]["fp8"] else x[_slots(st)]
    x = x.float()
    if scale is not None:
        x = x * scale.view(h, 1)
    return x.permute(0, 2, 1, 3)


def _visible(st, bits):
    """[sequences, rows, keys]; bits: [rows, bit] of the tree, None where rows stand in line."""
    w = st["case"]["window"]
    index, real = _padded(st)
    longest = index.shape[1]
    kv = st["seq_lens"].long().view(-1, 1, 1)
    n_q = (st["cu"][1:] - st["cu"][:-1]).long().view(-1, 1, 1)
    before = kv - n_q
    j = torch.arange(st["max_kv"], device="cuda").view(1, 1, -1)
    i = torch.arange(longest, device="cuda").view(1, -1, 1)
    if bits is None:
        row_pos, key_pos = before + i, j
        see = j <= row_pos
    else:
        b = bits[index][..., :longest] & real[:, None, :] & real[:, :, None]
        depth = b.sum(-1) - 1
        t = j - before
        inside = (t >= 0) & (t < n_q)
        t = t.clamp(0, longest - 1)
        see = (j < before) | (inside & torch.gather(b, 2, t.expand(-1, longest, -1)))
        row_pos = before + depth[:, :, None]
        key_pos = torch.where(j < before, j, before + torch.gather(depth, 1, t[:, 0])[:, None, :])
    if w:
        see = see & (row_pos - key_pos < w)
    return see & (j < kv) & real[:, :, None]


def _scores(st, bits=None):
    """Scaled scores of a padded batch, -inf where a row does not see a key:
    [sequences, kv heads, rows x group, keys], and the visibility."""
    case = st["case"]
    n, h = case["seqs"], case["kv_heads"]
    index, _ = _padded(st)
    q = st["q"][index].float().view(n, -1, h, GROUP, DIM).permute(0, 2, 1, 3, 4).reshape(n, h, -1, DIM)
    k = _gathered(st, st["k"], st.get("ks"))
    see = _visible(st, bits)
    s = torch.matmul(q, k.transpose(2, 3).contiguous())
    s *= SCALE
    rows = see.shape[1]
    s.view(n, h, rows, GROUP, -1).masked_fill_(~see[:, None, :, None, :], -math.inf)
    return s, see


def _plain_tree(st):
    case = st["case"]
    n, h = case["seqs"], case["kv_heads"]
    b = st["mask"]
    bits = ((b[:, :, None] >> torch.arange(64, device="cuda")) & 1).bool().reshape(b.shape[0], -1)
    s, _ = _scores(st, bits)
    rows = s.shape[2] // GROUP
    m = s.amax(-1, keepdim=True)
    sink = torch.full((h, GROUP), -math.inf, device="cuda") if st["sinks"] is None else st["sinks"].view(h, GROUP)
    sink = sink.view(1, h, 1, GROUP).expand(n, h, rows, GROUP).reshape(n, h, -1, 1)
    m = torch.maximum(m, sink)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)  # a row that sees nothing
    p = s.sub_(m).exp_()
    den = p.sum(-1, keepdim=True) + torch.exp(sink - m)
    o = torch.matmul(p, _gathered(st, st["v"], st.get("vs")).contiguous())
    o = torch.where(den > 0, o / den, torch.zeros_like(o))
    shape = lambda x: _rows(st, x.view(n, h, rows, GROUP, -1).permute(0, 2, 1, 3, 4).reshape(n, rows, h * GROUP, -1))
    out = shape(o).to(torch.bfloat16)
    return (out, shape(m + torch.log(den))[..., 0].contiguous()) if case["lse"] else out


def _plain_score(st):
    case = st["case"]
    n, h = case["seqs"], case["kv_heads"]
    s, _ = _scores(st)
    index, _ = _padded(st)
    lse = st["lse"][index].view(n, -1, h, GROUP).permute(0, 2, 1, 3).reshape(n, h, -1, 1)
    add = s.sub_(lse).exp_().sum(2)  # [sequences, kv heads, keys]
    at_s, at_j = _of_pairs(st["kv"], st["seq_lens"])
    page, place = st["table"].long()[at_s, at_j // PAGE], at_j % PAGE
    new = at_j >= (st["seq_lens"] - st["cu"][1:] + st["cu"][:-1])[at_s]
    old = st["scores"][page, :, place]
    st["scores"][page, :, place] = torch.where(new[:, None], torch.zeros_like(old), old) + add[at_s, :, at_j]
    return st["scores"]


def _plain_select(st):
    case = st["case"]
    n, h, budget = case["seqs"], case["kv_heads"], case["budget"]
    slots = _slots(st)
    left = st["seq_lens"].long().view(n, 1, 1)
    j = torch.arange(st["max_kv"], device="cuda").view(1, 1, -1)
    w = st["scores"][slots // PAGE, :, slots % PAGE].permute(0, 2, 1)
    w = torch.where((j < st["keep_first"]) | (j >= left - st["keep_last"]), torch.full_like(w, math.inf), w)
    w = torch.where(j < left, w, torch.full_like(w, -math.inf))
    best = w.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    best = torch.where(best < left, best, torch.full_like(best, 1 << 30)).sort(-1).values
    keep = torch.full((n, h, budget), -1, dtype=torch.int32, device="cuda")
    keep[..., : best.shape[-1]] = torch.where(best < left, best, torch.full_like(best, -1)).to(torch.int32)
    return keep, torch.clamp(st["seq_lens"], max=budget)


def _plain_move(st):
    case = st["case"]
    n, h = case["seqs"], case["kv_heads"]
    keep = st["keep"].long() if st["keep"].dim() == 3 else st["keep"].long()[:, None, :].expand(-1, h, -1)
    i = torch.arange(keep.shape[-1], device="cuda").view(1, 1, -1)
    start = st["starts"].long().view(n, 1, 1) if "starts" in st else torch.zeros((n, 1, 1), dtype=torch.int64, device="cuda")
    # (places behind the counts are marked -1: they repeat the sequence's first move)
    live = i < st["counts"].view(n, 1, 1)
    to = torch.where(live, start + i, start).expand_as(keep)
    keep = torch.where(live, keep, keep[..., :1])
    table, s = st["table"].long(), torch.arange(n, device="cuda").view(n, 1, 1)
    head = torch.arange(h, device="cuda").view(1, h, 1)
    slot = lambda row: table[s, row // PAGE] * PAGE + row % PAGE
    src, dst = slot(keep), slot(to)
    raw = torch.uint8 if case["fp8"] else torch.int16
    found = []
    for t in (st["k"], st["v"]):
        flat = t.view(raw).view(-1, st["pages"] * PAGE, h, DIM)
        flat[:, dst, head] = flat[:, src, head]
        found.append(t)
    if "scores" in st:
        w = st["scores"]
        w[dst // PAGE, head, dst % PAGE] = w[src // PAGE, head, src % PAGE]
        found.append(w)
    return tuple(found)


# ---- the package's calls --------------------------------------------------------------------

def _own(st):
    import eidola_amd as ea
    case = st["case"]
    h, op = case["kv_heads"], case["op"]
    geom = ea.AttnGeometry(num_q_heads=h * GROUP, num_kv_heads=h, softmax_scale=SCALE, window=case.get("window", 0),
                           kv_dtype=ea.KV_FP8_E4M3 if case.get("fp8") else ea.KV_BF16)
    if op == "tree":
        return ea.attn_tree(geom, st["q"], st["k"], st["v"], st["table"], st["seq_lens"], st["cu"], st["mask"],
                            max_q_len=max(st["q_lens"]), max_kv_len=st["max_kv"], sum_kv_len=st["sum_kv"],
                            sinks=st["sinks"], k_scale=st.get("ks"), v_scale=st.get("vs"), return_lse=case["lse"])
    if op == "score":
        return ea.kv_score(geom, st["q"], st["lse"], st["k"], st["table"], st["seq_lens"], st["cu"], st["scores"],
                           max_q_len=max(st["q_lens"]), max_kv_len=st["max_kv"], sum_kv_len=st["sum_kv"],
                           k_scale=st.get("ks"))
    if op == "select":
        return ea.kv_select(geom, st["scores"], st["table"], st["seq_lens"], budget=case["budget"],
                            keep_first=st["keep_first"], keep_last=st["keep_last"], max_kv_len=st["max_kv"])
    if op == "commit":
        ea.kv_compact(geom, st["layers_k"], st["layers_v"], st["table"], st["seq_lens"], st["keep"], st["counts"],
                      starts=st["starts"])
        return st["k"], st["v"]
    ea.kv_compact(geom, [st["k"]], [st["v"]], st["table"], st["seq_lens"], st["keep"], st["counts"],
                  scores=[st["scores"]])
    return st["k"], st["v"], st["scores"]


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state)
    return {"tree": _plain_tree, "score": _plain_score, "select": _plain_select, "commit": _plain_move,
            "compact": _plain_move}[op](state)


# ---- the definitions, in 64 bits ------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    n, h, op = case["seqs"], case["kv_heads"], case["op"]
    kv, q_lens = _lengths(case)
    w = case.get("window", 0)
    place = []  # slot of every token of a sequence
    for s in range(n):
        row = st["table"][s].long().repeat_interleave(PAGE)[: kv[s]] * PAGE
        place.append(row + torch.arange(kv[s], device="cuda") % PAGE)

    def rows_of(cache, scale, s):
        x = cache.reshape(-1, h, DIM).view(torch.uint8)[place[s]].view(torch.float8_e4m3fn).double() \
            if case["fp8"] else cache.reshape(-1, h, DIM)[place[s]].double()
        return x if scale is None else x * scale.double()[None, :, None]

    if op == "tree":
        outs, lses, at = [], [], 0
        for s in range(n):
            up = _parents(case, s, seed)
            t, before = len(up), kv[s] - len(up)
            see = torch.zeros((t, kv[s]), dtype=torch.bool)
            depth = []
            for i, u in enumerate(up):
                depth.append(depth[u] + 1 if u >= 0 else 0)
                see[i] = see[u] if u >= 0 else torch.arange(kv[s]) < before
                see[i, before + i] = True
            if w:
                key = torch.cat([torch.arange(before), before + torch.tensor(depth)])
                see &= (before + torch.tensor(depth))[:, None] - key[None, :] < w
            see = see.cuda()
            k, v = rows_of(st["k"], st.get("ks"), s), rows_of(st["v"], st.get("vs"), s)
            o = torch.empty((t, h * GROUP, DIM), dtype=torch.float64, device="cuda")
            l = torch.empty((t, h * GROUP), dtype=torch.float64, device="cuda")
            for c in range(h * GROUP):
                x = st["q"][at:at + t, c].double() @ k[:, c // GROUP].t().contiguous() * SCALE
                x = x.masked_fill(~see, -math.inf)
                if case["sinks"]:
                    x = torch.cat([x, st["sinks"][c].double().expand(t, 1)], 1)
                l[:, c] = torch.logsumexp(x, 1)
                o[:, c] = torch.softmax(x, 1)[:, : kv[s]] @ v[:, c // GROUP]
            outs.append(o)
            lses.append(l)
            at += t
        return (torch.cat(outs), torch.cat(lses)) if case["lse"] else torch.cat(outs)
    if op == "score":
        table, at = st["scores"].double(), 0
        for s in range(n):
            t = q_lens[s]
            k = rows_of(st["k"], st.get("ks"), s)
            pos = torch.arange(kv[s] - t, kv[s], device="cuda")[:, None]
            key = torch.arange(kv[s], device="cuda")[None, :]
            see = (key <= pos) & (key > pos - w) if w else key <= pos
            table[place[s][kv[s] - t:] // PAGE, :, place[s][kv[s] - t:] % PAGE] = 0
            for c in range(h * GROUP):
                x = st["q"][at:at + t, c].double() @ k[:, c // GROUP].t().contiguous() * SCALE
                p = torch.exp(x - st["lse"][at:at + t, c].double()[:, None]).masked_fill(~see, 0).sum(0)
                table[place[s] // PAGE, c // GROUP, place[s] % PAGE] += p
            at += t
        return table
    if op == "select":
        return None  # (whole numbers)
    # rows are moved as they stand: one sequence and head after the other, from a copy
    raw = torch.uint8 if case["fp8"] else torch.int16
    found = []
    for name in ("k", "v"):
        new = st[name].view(raw).view(-1, st["pages"] * PAGE, h, DIM).clone()
        old = new.clone()
        for s in range(n):
            m = int(st["counts"][s])
            first = int(st["starts"][s]) if "starts" in st else 0
            for c in range(h):
                rows = st["keep"][s, :m] if st["keep"].dim() == 2 else st["keep"][s, c, :m]
                new[:, place[s][first:first + m], c] = old[:, place[s][rows.long()], c]
        found.append(new.view(st[name].dtype).view(st[name].shape).float().double())
    if "scores" in st:
        new, old = st["scores"].double(), st["scores"].double()
        for s in range(n):
            m = int(st["counts"][s])
            for c in range(h):
                a, b = place[s][:m], place[s][st["keep"][s, c, :m].long()]
                new[a // PAGE, c, a % PAGE] = old[b // PAGE, c, b % PAGE]
        found.append(new)
    return tuple(found)
