"""eid_kv_score where rows or keys are not ordinary numbers, and where many parts are joined."""
import numpy as np
import pytest
import torch

import eidola_amd as ea
from eidola_amd import KV_BF16, KV_FP8_E4M3, synth

import cache_ref as R
from test_gpu_cache_rows import G, REL, lse_of, pool, score  # noqa: F401 (G: fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("heads", [2, 8])
@pytest.mark.parametrize("q_lens", [[1, 1, 2], [1, 5, 2], [1, 40, 3]])
def test_rows_that_do_not_exist_or_saw_nothing_add_nothing_beside_infinite_keys(G, q_lens, heads, window):
    # A key of -inf in one element where every row is positive: its scores are -inf, its weights 0.  Rows whose
    # lse says that they saw nothing add nothing even to a key that is NaN.
    b, q, kc, vc, ks, vs, sinks = R.filled([200, 90, 33], q_lens, num_kv_heads=heads, window=window)
    q[:, :, 5] = 0x3F80
    kc.reshape(-1, heads, 64)[b.all_slots(0)[190], :, 5] = 0xFF80
    kc.reshape(-1, heads, 64)[b.all_slots(1)[60], :, 5] = 0xFF80
    kc.reshape(-1, heads, 64)[b.all_slots(2)[20], :, 5] = 0x7FC0
    lse = lse_of(b, q, kc, vc, sinks, ks, vs)
    lse[b.cu_seqlens_q[2]:] = -np.inf
    if q_lens[1] > 3:
        lse[b.cu_seqlens_q[1] + 2, ::3] = -np.inf
    w = pool(b, np.random.default_rng(1))
    ref = R.kv_score(b, q, lse, kc, w, ks)
    assert np.isfinite(ref).all()
    got = score(G, b, q, lse, kc, w, ks)
    assert (np.abs(got - ref) <= REL * ref + 1e-7).all()


@pytest.mark.parametrize("kv_dtype", [KV_BF16, KV_FP8_E4M3])
@pytest.mark.parametrize("window", [0, 1, 100])
def test_many_parts_are_joined(G, window, kv_dtype):
    # 18 parts.  A sum has up to 8 x 300 terms: 2400 * 2^-24 = 1.43e-4 of it, beside the exponents' 1.2e-5 and the
    # scores' 2.3e-5: 1.8e-4 in all.
    b, q, kc, vc, ks, vs, sinks = R.filled([700], [300], num_kv_heads=2, window=window, kv_dtype=kv_dtype)
    desc = ea.make_desc(b.geom, num_seqs=1, num_q_tokens=300, max_q_len=300, max_kv_len=700,
                        max_blocks_per_seq=b.block_table.shape[1], num_blocks=b.num_blocks)
    assert ea.kv_score_workspace_bytes(desc) >= 16 * 2 * 700 * 4
    lse = lse_of(b, q, kc, vc, sinks, ks, vs)
    w = pool(b, np.random.default_rng(3))
    ref = R.kv_score(b, q, lse, kc, w, ks)
    got = score(G, b, q, lse, kc, w, ks)
    assert (np.abs(got - ref) <= 1.8e-4 * ref + 1e-7).all()
    assert np.array_equal(got, score(G, b, q, lse, kc, w, ks))


@pytest.mark.parametrize("kv_dtype", [KV_BF16, KV_FP8_E4M3])
@pytest.mark.parametrize("heads,seqs", [(1, 5), (2, 90), (8, 3)])
def test_chunks_beside_short_sequences_share_one_line_of_tiles(G, heads, seqs, kv_dtype):
    # long chunks first, in the middle and last, their sums in a workspace that follows the batch's keys; also with
    # a descriptor that says less than there is, for which no place is left.  Up to 8 x 70 terms per sum:
    # 560 * 2^-24 = 3.4e-5 of it, beside the exponents' 1.2e-5 and the scores' 2.3e-5: 7e-5 in all.
    rng = np.random.default_rng(seqs)
    q_lens = rng.choice([1, 2, 3, 7], seqs)
    seq_lens = np.array([int(rng.integers(n, 150)) for n in q_lens])
    for i in (0, seqs // 2, seqs - 1):
        q_lens[i], seq_lens[i] = 70 - i % 3, 1100 + i
    b, q, kc, vc, ks, vs, sinks = R.filled(seq_lens, q_lens, num_kv_heads=heads, kv_dtype=kv_dtype)
    lse = lse_of(b, q, kc, vc, sinks, ks, vs)
    w = pool(b, rng)
    ref = R.kv_score(b, q, lse, kc, w, ks)
    for total in (0, int(seq_lens.sum()), int(seq_lens.max())):
        desc = ea.make_desc(b.geom, num_seqs=seqs, num_q_tokens=len(q), max_q_len=b.max_q_len, max_kv_len=b.max_kv_len,
                            max_blocks_per_seq=b.block_table.shape[1], num_blocks=b.num_blocks, sum_kv_len=total)
        need = ea.kv_score_workspace_bytes(desc)
        assert total == 0 or need > 0
        guard = 1 << 16                                   # what lies behind the workspace stays as it is
        ws = torch.full((need + guard,), 255, dtype=torch.uint8, device="cuda")
        got = score(G, b, q, lse, kc, w, ks, sum_kv_len=total, workspace=ws[:need] if need else ws)
        assert (np.abs(got - ref) <= 7e-5 * ref + 1e-7).all()
        assert bool((ws[need:] == 255).all())
