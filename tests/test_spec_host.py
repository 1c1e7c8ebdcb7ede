"""CPU: the speculative-step operators' host side -- rotary frequencies against
their published formulas, workspace sizes, and every refusal (arguments are
checked before the device, so a refused call touches no GPU)."""
import ctypes as C
import math

import numpy as np
import pytest

import kanjoos_amd as K

F32, F16, BF16 = K.TYPE_F32, K.TYPE_F16, K.TYPE_BF16
A = 1 << 20  # an aligned address that no refused call reads


def refused(call, match, code=K.KNJ_E_ARG):
    with pytest.raises(K.KnjError, match=match) as e:
        call()
    assert e.value.code == code


# ------------------------------------------------------------------ rotary frequencies

@pytest.mark.parametrize("n,base", [(8, 1e4), (64, 1e4), (96, 5e5), (128, 1e6)])
def test_rope_freqs(n, base):
    i = np.arange(n // 2)
    plain = base ** (-2.0 * i / n)
    f, ms = K.rope_freqs(n, base)
    np.testing.assert_allclose(f, plain, rtol=1e-15)
    assert ms == 1.0
    f, ms = K.rope_freqs(n, base, K.ROPE_LINEAR, 4.0)
    np.testing.assert_allclose(f, plain / 4, rtol=1e-15)
    f, ms = K.rope_freqs(n, base, K.ROPE_NTK, 4.0)
    # the slowest pair is slowed by the factor, the fastest is kept
    np.testing.assert_allclose(f[[0, -1]], [1.0, plain[-1] / 4], rtol=1e-12)


def test_rope_freqs_yarn():
    """Pairs that turn more than 32 times in the original context are kept, those
    that turn less than once are divided, and the ramp between is linear in i."""
    n, base, ctx, s = 128, 1e6, 32768, 4.0
    plain = base ** (-2.0 * np.arange(n // 2) / n)
    f, ms = K.rope_freqs(n, base, K.ROPE_YARN, s, ctx)
    assert ms == np.float32(0.1 * math.log(s) + 1)
    turns = ctx * plain / (2 * math.pi)
    keep = (f / plain - 1 / s) / (1 - 1 / s)
    # (numpy's powers and the library's may part by an ulp, 2e-16, amplified here by s / (s - 1))
    assert np.all(np.abs(keep[turns > 40] - 1) < 1e-12) and np.all(np.abs(keep[turns < 0.7]) < 1e-12)
    ramp = keep[(keep > 1e-9) & (keep < 1 - 1e-9)]
    assert ramp.size > 5
    np.testing.assert_allclose(np.diff(ramp), np.diff(ramp)[0], rtol=1e-9)


def test_rope_freqs_llama3():
    n, base, ctx, s = 128, 5e5, 8192, 8.0
    plain = base ** (-2.0 * np.arange(n // 2) / n)
    f, ms = K.rope_freqs(n, base, K.ROPE_LLAMA3, s, ctx)
    assert ms == 1.0
    wave = 2 * math.pi / plain
    for fi, pi, wi in zip(f, plain, wave):
        if wi < ctx / 4:
            want = pi
        elif wi > ctx / 1:
            want = pi / s
        else:
            k = (ctx / wi - 1) / (4 - 1)
            want = (1 - k) * pi / s + k * pi
        assert fi == pytest.approx(want, rel=1e-12)


@pytest.mark.parametrize("kw,match", [
    (dict(n_rot=0), "n_rot"), (dict(n_rot=12), "n_rot"), (dict(n_rot=136), "n_rot"), (dict(base=1.0), "base"),
    (dict(base=math.inf), "base"), (dict(scaling=5), "scaling"), (dict(scaling=-1), "scaling"),
    (dict(scaling=K.ROPE_LINEAR, factor=0.5), "factor"), (dict(scaling=K.ROPE_NTK, factor=math.nan), "factor"),
    (dict(scaling=K.ROPE_YARN, factor=2.0), "yarn"), (dict(scaling=K.ROPE_YARN, factor=2.0, orig_ctx=4096, p0=1, p1=2), "yarn"),
    (dict(scaling=K.ROPE_LLAMA3, factor=2.0, orig_ctx=4096, p0=4, p1=4), "llama3")])
def test_rope_freqs_refusals(kw, match):
    refused(lambda: K.rope_freqs(**{**dict(n_rot=64, base=1e4), **kw}), match)


# ------------------------------------------------------------------ refusals

@pytest.mark.parametrize("kw,match", [
    (dict(type_id=K.TYPE_Q4_K), "activations"), (dict(layout=2), "layout"), (dict(head_dim=96), "head_dim"),
    (dict(n_rot=4), "n_rot"), (dict(n_rot=136), "n_rot"), (dict(q=None), "null"), (dict(pos=None), "null"),
    (dict(inv_freq=None), "null"), (dict(q_out=None, q=None), "null"), (dict(k=None, k_out=A), "null"),
    (dict(n_rows=-1), "row count"), (dict(n_head=0), "n_head"), (dict(q_stride=1016), "stride"),
    (dict(k_stride=120), "stride"), (dict(q=A + 4), "16-byte"), (dict(q_stride=1026), "16-byte"),
    (dict(type_id=F16, q_out=A, q_out_stride=1028), "16-byte"), (dict(mscale=0.0), "mscale"),
    (dict(mscale=math.inf), "mscale"), (dict(q_norm=A + 4), "aligned"), (dict(inv_freq=A + 4), "aligned")])
def test_rope_refusals(kw, match):
    a = dict(type_id=F32, q=A, k=A, pos=A, inv_freq=A, n_rows=4, n_head=8, n_head_kv=1, head_dim=128)
    refused(lambda: K.rope(**{**a, **kw}), match)


def cache(**kw):
    a = dict(format=K.KV_I8, n_seq=2, n_head_kv=4, n_ctx=100, head_dim=128, k=A, v=A, k_scale=A, v_scale=A, seq_stride=0)
    return K.KvCache(**{**a, **kw})


BAD_CACHES = [(dict(format=3), "format"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(k_scale=None), "k_scale"),
              (dict(v_scale=None, format=K.KV_F8), "k_scale"), (dict(head_dim=80), "head_dim"), (dict(n_seq=0), "n_seq"),
              (dict(n_head_kv=65), "n_head_kv"), (dict(n_head_kv=0), "n_head_kv"), (dict(n_ctx=0), "n_ctx"),
              (dict(seq_stride=4 * 100 * 128 - 128), "seq_stride"), (dict(seq_stride=4 * 100 * 128 + 64), "seq_stride"),
              (dict(k=A + 8), "16-byte"), (dict(v_scale=A + 2), "4-byte")]


@pytest.mark.parametrize("kw,match", BAD_CACHES)
def test_cache_refusals(kw, match):
    c = cache(**kw)
    refused(lambda: K.kv_store(c, F32, A, A, A, 1, row_stride=512), match)
    refused(lambda: K.kv_load(c, F32, A, A, 1, row_stride=512), match)
    refused(lambda: K.attention_tree(c, F32, A, A, 32, 1, A, 8, q_stride=4096, out_stride=4096), match)
    assert K.attention_tree_workspace(c, 32, 1, 8) == 0


@pytest.mark.parametrize("kw,match", [
    (dict(type_id=K.TYPE_Q6_K), "activations"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(n_rows=-1), "row count"),
    (dict(row_stride=508), "stride"), (dict(row_stride=513), "16-byte"), (dict(v=A + 8), "16-byte"),
    (dict(n_rows=2 ** 31 - 1), "too many")])
def test_kv_row_refusals(kw, match):
    a = dict(cache=cache(), type_id=F32, k=A, v=A, n_rows=3, row_stride=512)
    refused(lambda: K.kv_load(**{**a, **kw}), match)
    refused(lambda: K.kv_store(**{**a, "start": A, **kw}), match)
    refused(lambda: K.kv_store(**{**a, "start": None}), "null start")
    assert K.lib().knj_kv_store(None, F32, A, A, 512, A, None, 1, None) == K.KNJ_E_ARG
    assert K.lib().knj_attention_tree_workspace(None, 8, 1, 1) == 0


class Workspace:
    """Stands in for a DeviceBuffer that is never read."""

    def __init__(self, nbytes):
        self.nbytes = nbytes


@pytest.mark.parametrize("kw,match", [
    (dict(type_id=12), "activations"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(prefix=None), "null"),
    (dict(n_rows=-1), "n_rows"), (dict(n_rows=1025, max_prefix=0), "n_rows"), (dict(n_head=30), "multiple"),
    (dict(n_head=0), "multiple"), (dict(max_prefix=-1), "n_ctx"), (dict(max_prefix=2 ** 31 - 1), "n_ctx"),
    (dict(max_prefix=1990, n_rows=11), "n_ctx"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"), (dict(q_stride=4088), "stride"),
    (dict(out_stride=4088), "stride"), (dict(q_stride=4098), "16-byte"), (dict(out=A + 8), "16-byte"),
    (dict(), "workspace of")])
def test_attention_tree_refusals(kw, match):
    a = dict(cache=cache(n_ctx=2000), type_id=F32, q=A, out=A, n_head=32, n_rows=3, prefix=A, max_prefix=1900)
    refused(lambda: K.attention_tree(**{**a, **kw}), match)


def test_attention_tree_workspace_size():
    """A short workspace is refused with the size that knj_attention_tree_workspace
    returns; a misaligned one too."""
    c = cache(n_ctx=2000)
    need = K.attention_tree_workspace(c, 32, 3, 1900)
    assert need > 0
    L = K.lib()

    def call(ws, nbytes):
        return L.knj_attention_tree(c.ref, F32, A, 4096, 32, 3, A, 1900, None, None, 0, 0.1, A, 4096, ws, nbytes, None)

    assert call(A, need - 1) == K.KNJ_E_ARG
    assert str(need).encode() in L.knj_last_error()
    assert call(A + 8, need) == K.KNJ_E_ARG
    for bad in [(31, 3, 1900), (0, 3, 1900), (32, 0, 1900), (32, 1025, 0), (32, 3, -1), (32, 3, 1998)]:
        assert K.attention_tree_workspace(c, *bad) == 0


@pytest.mark.parametrize("kw,match", [
    (dict(type_id=14), "logits must"), (dict(logits=None), "null"), (dict(logits=A + 2), "aligned"),
    (dict(type_id=BF16, logits=A + 1), "aligned"), (dict(n_rows=-1), "row count"), (dict(n_vocab=0), "n_vocab"),
    (dict(n_vocab=(1 << 20) + 1), "n_vocab"), (dict(row_stride=999), "stride"), (dict(temperature=0.0), "temperature"),
    (dict(temperature=-1.0), "temperature"), (dict(temperature=math.nan), "temperature"), (dict(temperature=math.inf), "temperature"),
    (dict(tokens=A), "together"), (dict(logprob=A), "together"), (dict(n_top=33), "n_top"), (dict(n_top=-1), "n_top"),
    (dict(n_top=5, n_vocab=4), "n_top"), (dict(n_top=2), "top_idx"), (dict(n_top=2, top_idx=A), "top_idx"),
    (dict(n_rows=2 ** 31 - 1, n_vocab=5000), "too many"), (dict(), "workspace of")])
def test_token_logprobs_refusals(kw, match):
    a = dict(type_id=F32, logits=A, n_rows=7, n_vocab=1000, workspace=None)
    refused(lambda: K.token_logprobs(**{**a, **kw}), match)


@pytest.mark.parametrize("n_rows,n_vocab", [(1 << 24, 8), (1 << 23, 20000)])
def test_token_logprobs_row_limits(n_rows, n_vocab):
    """A launch holds 2^32 threads along a dimension of its grid: 256 a row, 64 a piece."""
    L = K.lib()
    assert L.knj_token_logprobs(F32, A, n_vocab, n_rows, n_vocab, 1.0, None, None, A, 0, None, None, A,
                                K.token_logprobs_workspace(n_rows, n_vocab), None) == K.KNJ_E_ARG
    assert b"too many" in L.knj_last_error()


def test_row_limits():
    refused(lambda: K.rope(F32, A, A, A, A, 1 << 24, 8, 1, 128), "too many")
    c = cache(n_ctx=1 << 25)
    n = (1 << 27) // c.desc.n_head_kv
    refused(lambda: K.kv_store(c, F32, A, A, A, n), "too many")
    refused(lambda: K.kv_load(c, F32, A, A, n), "too many")


@pytest.mark.parametrize("n_head,n_seq", [(2, 1), (8, 1), (32, 1), (32, 5), (64, 65535)])
def test_attention_tree_workspace_bound(n_head, n_seq):
    """No sizes need more than the documented 262144 (head_dim + 4) bytes."""
    for n_head_kv, head_dim in ((1, 64), (2, 128)):
        c = cache(n_head_kv=n_head_kv, head_dim=head_dim, n_seq=n_seq, n_ctx=1 << 22)
        for n_rows in (1, 2, 7, 16, 33, 64, 100, 257, 1024):
            for prefix in (0, 1, 100, 1000, 4096, 50000, (1 << 22) - 1024):
                need = K.attention_tree_workspace(c, n_head, n_rows, prefix)
                assert need <= 262144 * (head_dim + 4)


def test_token_logprobs_workspace_size():
    need = K.token_logprobs_workspace(7, 5000)
    assert need > 0 and K.token_logprobs_workspace(14, 5000) == 2 * need
    assert [K.token_logprobs_workspace(*b) for b in [(0, 10), (3, 0), (3, (1 << 20) + 1), (-1, 10)]] == [0] * 4
    L = K.lib()
    assert L.knj_token_logprobs(F32, A, 5000, 7, 5000, 1.0, None, None, A, 0, None, None, A, need - 1, None) == K.KNJ_E_ARG
    assert str(need).encode() in L.knj_last_error()
    assert L.knj_token_logprobs(F32, A, 5000, 7, 5000, 1.0, None, None, A, 0, None, None, A + 4, need, None) == K.KNJ_E_ARG


def test_valid_calls_need_an_open_device():
    """Correct arguments reach the device check: refused before knj_device_open,
    with nothing launched (a call of no rows included)."""
    c = cache()
    ws = Workspace(1 << 30)
    L = K.lib()
    if L.knj_synchronize() == K.KNJ_OK:
        pytest.skip("a GPU is present")
    for call in (lambda: K.rope(F32, A, A, A, A, 4, 8, 1, 128), lambda: K.rope(F32, A, A, A, A, 0, 8, 1, 128),
                 lambda: K.kv_store(c, F32, A, A, A, 1), lambda: K.kv_load(c, F32, A, A, 0)):
        refused(call, "not open", K.KNJ_E_STATE)
    assert L.knj_attention_tree(c.ref, F32, A, 4096, 32, 3, A, 90, None, None, 0, 0.1, A, 4096, A, ws.nbytes,
                                None) == K.KNJ_E_STATE
    assert L.knj_token_logprobs(F32, A, 10, 7, 10, 1.0, None, None, A, 0, None, None, A, ws.nbytes, None) == K.KNJ_E_STATE
