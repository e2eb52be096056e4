"""Sizes at the end of what the tree attention and the operators over cached rows take: host code, no GPU."""
import ctypes as C

import pytest

import eidola_amd as ea
from eidola_amd import _lib

from test_cache_ops_abi import args, desc, tree

UNSUP = _lib.EID_ERR_UNSUPPORTED
ROWS = 0x7FFF0000       # longest sequence: the kernels look up to 64 Ki rows past its end in 32 bits


@pytest.mark.parametrize("over", [1, 0xFFFF])
def test_sequences_whose_rows_would_not_be_counted_in_32_bits_are_refused(over):
    # (accepted, they would be read and written at wrapped indices)
    lib, ok = ea.load_library(), 0x1000
    d = desc(num_seqs=1, max_kv_len=ROWS + over, max_blocks_per_seq=(ROWS + over + 15) // 16)
    assert ea.attn_tree_workspace_bytes(d) == 0 and ea.kv_score_workspace_bytes(d) == 0
    assert tree(d, args(d)) == UNSUP
    assert lib.eid_kv_score(C.byref(d), ok, ok, ok, ok, ok, ok, None, ok, None, 0, None) == UNSUP
    assert lib.eid_kv_select(C.byref(d), ok, ok, ok, 64, 4, 16, ok, ok, None) == UNSUP
    one = (C.c_int64 * 1)(ok)
    assert lib.eid_kv_compact(C.byref(d), 1, one, one, None, ok, ok, ok, 0, 8, 0, 8, ok, None, None) == UNSUP


def test_the_longest_sequences_are_planned():
    d = desc(num_seqs=1, max_kv_len=ROWS, max_blocks_per_seq=ROWS // 16)
    assert 0 < ea.attn_tree_workspace_bytes(d) <= 256 << 20


def test_the_workspace_of_scores_does_not_grow_with_what_a_ragged_batch_could_hold():
    # one long chunk beside many short sequences: the bound follows the keys, not sequences x longest
    for heads, seqs, rows, longest in ((1, 256, 512, 131072), (1, 64, 2048, 131072), (8, 32, 512, 32768), (2, 1000, 300, 70000)):
        geom = ea.AttnGeometry(num_q_heads=8 * heads, num_kv_heads=heads)
        d = ea.make_desc(geom, num_seqs=seqs, num_q_tokens=rows + seqs - 1, max_q_len=rows, max_kv_len=longest,
                         max_blocks_per_seq=(longest + 15) // 16, num_blocks=longest, sum_kv_len=longest + 100 * seqs)
        assert ea.kv_score_workspace_bytes(d) <= 4 << 20
        d.sum_kv_len = 0
        assert ea.kv_score_workspace_bytes(d) <= 4 << 20
