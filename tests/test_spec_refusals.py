"""CPU: calls of the speculative-step operators whose arguments would give wrong
results or pass what the kernels index, refused before any device is touched."""
import math

import pytest

import kanjoos_amd as K
from test_spec_host import A, F32, cache, refused


@pytest.mark.parametrize("eps", [-1e-6, math.nan, math.inf])
def test_rope_eps(eps):
    """Of a norm; a call without norms does not read it."""
    for norms in (dict(q_norm=A), dict(k_norm=A)):
        refused(lambda: K.rope(F32, A, A, A, A, 4, 8, 1, 128, eps=eps, **norms), "eps")
    if K.lib().knj_synchronize() != K.KNJ_OK:  # (no GPU: the next check is the device's)
        refused(lambda: K.rope(F32, A, A, A, A, 4, 8, 1, 128, eps=eps), "not open", K.KNJ_E_STATE)


def test_in_place_with_another_stride():
    """Rows written over rows that are still to be read."""
    a = dict(type_id=F32, q=A, k=2 * A, pos=A, inv_freq=A, n_rows=4, n_head=8, n_head_kv=1, head_dim=128)
    refused(lambda: K.rope(**{**a, "q_out": A, "q_stride": 1536}), "in place")  # (q_out_stride defaults to packed rows)
    refused(lambda: K.rope(**{**a, "k_out": 2 * A, "k_stride": 1536, "k_out_stride": 256}), "in place")
    c = cache(n_ctx=200)
    for n_seq, n_rows in ((2, 1), (1, 3)):
        c = cache(n_ctx=200, n_seq=n_seq)
        refused(lambda: K.attention_tree(c, F32, A, A, 32, n_rows, A, 100, q_stride=5120), "in place")
    if K.lib().knj_synchronize() != K.KNJ_OK:  # one row has no other to overwrite
        refused(lambda: K.rope(**{**a, "q_out": A, "q_stride": 1536, "n_rows": 1}), "not open", K.KNJ_E_STATE)


def test_attention_tree_slot_limit():
    """Slots are numbered in 32 bits, with a chunk that is fetched past the last one."""
    c = cache(n_ctx=2 ** 31 - 1, n_seq=1, n_head_kv=1, head_dim=64)
    most = 2 ** 31 - 1 - 256
    for n_rows in (1, 1000):
        assert 0 < K.attention_tree_workspace(c, 8, n_rows, most - n_rows) <= 262144 * 68
        for over in (1, 200, 256):
            assert K.attention_tree_workspace(c, 8, n_rows, most - n_rows + over) == 0
            refused(lambda: K.attention_tree(c, F32, A, A, 8, n_rows, A, most - n_rows + over), "2\\^31")


@pytest.mark.parametrize("off", [1, 2, 3])
def test_misaligned_arrays(off):
    """Lengths, slots, masks and outputs off their types' boundaries (a scalar load
    would drop the address's low bits)."""
    bad, c = A + off, cache(n_ctx=200)
    refused(lambda: K.rope(F32, A, A, bad, A, 4, 8, 1, 128), "pos must")
    refused(lambda: K.kv_store(c, F32, A, A, bad, 1), "start")
    refused(lambda: K.kv_store(c, F32, A, A, A, 1, counts=bad), "counts")
    refused(lambda: K.kv_load(c, F32, A, A, 1, slots=bad), "slots")
    refused(lambda: K.attention_tree(c, F32, A, 2 * A, 32, 1, bad, 100), "prefix")
    refused(lambda: K.attention_tree(c, F32, A, 2 * A, 32, 1, A, 100, counts=bad), "counts")
    refused(lambda: K.attention_tree(c, F32, A, 2 * A, 32, 1, A, 100, mask=A + 4), "mask")
    for kw in (dict(tokens=bad, logprob=A), dict(tokens=A, logprob=bad), dict(entropy=bad), dict(n_top=2, top_idx=bad, top_logprob=A),
               dict(n_top=2, top_idx=A, top_logprob=bad)):
        refused(lambda: K.token_logprobs(F32, A, 7, 1000, None, **kw), "aligned")
