"""CPU: the 4-bit pages' sizes and refusals, and the numpy model that the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import kanjoos_amd as K
from pages_model import Pool, groups, half, row_bytes, values
from test_spec_host import A, F16, F32, Workspace, refused


def pages(**kw):
    a = dict(n_layer=2, n_page=10, page_size=32, n_head_kv=4, head_dim=128, n_seq=3, n_table=4, data=A, table=A, refs=A)
    return K.KvPages(**{**a, **kw})


# ------------------------------------------------------------------ the model

def test_groups_round_as_stated():
    """A code's value is at most half a step off, and the step at most (largest - low) / 15 of f16's next."""
    rng = np.random.default_rng(0)
    x = rng.normal(size=(500, 128)) * np.exp(3 * rng.normal(size=(500, 1)))
    code, step, low = groups(x)
    v = values(code, step, low)
    g = x.reshape(500, 4, 32)
    assert np.all(step <= np.maximum((g.max(-1) - low) / 15, 0)) and np.all(half(step) == step) and np.all(half(low) == low)
    # half a step inside the 16 levels, and above the last what the step's rounding leaves (15 * 2^-10 of it, or
    # of a step below 2^-14 15 units of 2^-24); f16's rounding of the value
    slack = np.maximum(0.5, 15 * 2.0 ** -10) * step + 15 * 2.0 ** -24 + 2.0 ** -10 * np.abs(g).max(-1)
    assert np.all(np.abs(v.reshape(g.shape) - g) <= slack[..., None])
    assert code.max() == 15 and code.min() == 0


def test_groups_of_no_range_and_not_held():
    x = np.zeros((6, 64))
    x[0] = 3.14159
    x[1, :32] = np.linspace(0, 14 * 2.0 ** -24, 32)  # a range below 15 of f16's least
    x[2, 5], x[3, 6], x[4, 7], x[5, 8] = np.inf, np.nan, 65505.0, -65504.0
    code, step, low = groups(x)
    assert np.all(code[1] == 0) and np.all(step[1] == 0)
    assert np.isnan(low[2:5, 0]).all() and np.all(low[2:5, 1] == 0)
    v = values(code, step, low)
    assert np.all(v[0] == half(np.float64(3.14159))) and np.isnan(v[2:5, :32]).all()
    assert abs(v[5, 8] + 65504) <= 32 and np.all(np.abs(v[5]) < 65520)


def test_bytes_hold_the_codes_in_order():
    x = np.arange(32.0) / 31 * 15
    code, step, _ = groups(x)
    words, meta = row_bytes(x)
    w = words.view(np.uint32)
    got = [(int(w[d // 8]) >> (4 * (d % 8 // 2) + 16 * (d % 2))) & 15 for d in range(32)]
    assert got == code[0].tolist()
    assert meta.view(np.float16)[0] == step[0] and meta.view(np.float16)[1] == 0


# ------------------------------------------------------------------ sizes and refusals

@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 256])
def test_bytes(D, page):
    p = pages(head_dim=D, page_size=page, data=None, table=None, refs=None)
    rng = np.random.default_rng(0)
    assert K.lib().knj_pages_bytes(p.ref) == Pool(rng, 2, 10, page, 4, D, 3, 4).data.nbytes
    assert K.pages_workspace(p) >= 4 * 3 * 4
    big = pages(n_layer=48, n_page=2 ** 26 - 1, n_head_kv=64, page_size=256)
    assert K.lib().knj_pages_bytes(big.ref) == 48 * (2 ** 26 - 1) * 64 * 256 * 160


SIZES = [(dict(head_dim=96), "head_dim"), (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"),
         (dict(page_size=512), "page_size"), (dict(n_head_kv=0), "n_head_kv"), (dict(n_head_kv=65), "n_head_kv"),
         (dict(n_layer=0), "n_layer"), (dict(n_layer=1025), "n_layer"), (dict(n_page=0), "n_page"), (dict(n_page=2 ** 26), "n_page"),
         (dict(n_seq=0), "n_seq"), (dict(n_seq=4097), "n_seq"), (dict(n_table=0), "n_table"), (dict(n_table=2 ** 26), "n_table"),
         (dict(n_seq=4096, n_table=2 ** 20), "entries")]
POINTERS = [(dict(data=None), "null"), (dict(data=A + 8), "16-byte"), (dict(table=A + 2), "aligned"), (dict(refs=A + 1), "aligned")]


def every_call(p):
    ws = Workspace(2 ** 40)
    ws.ptr = A
    lib, s = K.lib(), None
    return [lambda: K.pages_store(p, 0, F32, A, A, A, 1, row_stride=8192), lambda: K.pages_load(p, 0, F32, A, A, 1, row_stride=8192),
            lambda: K.attention_pages(p, 0, F32, A, 2 * A, 128, 1, A, 8, q_stride=16384, out_stride=16384),
            lambda: K.check(lib.knj_pages_reserve(p.ref, s, A, A, A, A, 2 ** 40, s)),
            lambda: K.check(lib.knj_pages_fork(p.ref, A, s, A, 2 ** 40, s)), lambda: K.pages_free(p, A),
            lambda: K.pages_compact(p, A, A, 1), lambda: K.pages_copy(p, pages(), A, A, 1), lambda: K.pages_copy(pages(), p, A, A, 1)]


@pytest.mark.parametrize("kw,match", SIZES + POINTERS)
def test_pool_refusals(kw, match):
    p = pages(**kw)
    for call in every_call(p):
        refused(call, match)
    if (kw, match) in SIZES:
        assert K.lib().knj_pages_bytes(p.ref) == 0 and K.pages_workspace(p) == 0
        assert K.attention_pages_workspace(p, 128, 1, 8) == 0
        if "n_seq" not in kw or kw["n_seq"] <= 4096:
            with pytest.raises(K.KnjError):
                K.KvPages.allocate(**{n: getattr(p.desc, n) for n in ("n_layer", "n_page", "page_size", "n_head_kv", "head_dim",
                                                                      "n_seq", "n_table")})
    for f in ("knj_pages_bytes", "knj_pages_workspace"):
        assert getattr(K.lib(), f)(None) == 0


def test_most_entries():
    """Entries are counted in 32 bits, 1024 at a time: a table whose last step would pass 2^31 is refused."""
    def kw(entries, n_seq):
        return dict(n_seq=n_seq, n_table=entries // n_seq, n_page=2 ** 20, page_size=16)
    most = pages(**kw(2 ** 31 - 1025, 3729))
    assert most.desc.n_seq * most.desc.n_table == 2 ** 31 - 1025
    assert K.lib().knj_pages_bytes(most.ref) > 0 and K.pages_workspace(most) > 0
    for entries, n_seq in ((2 ** 31 - 1024, 4064), (2 ** 31 - 128, 4095), (2 ** 31 - 512, 4094)):
        p = pages(**kw(entries, n_seq))
        assert p.desc.n_seq * p.desc.n_table == entries
        for call in every_call(p):
            refused(call, "entries")
        assert K.lib().knj_pages_bytes(p.ref) == 0 and K.pages_workspace(p) == 0


def test_missing_tables():
    for call in every_call(pages(table=None))[:-2]:
        refused(call, "null")
    for call in every_call(pages(refs=None))[3:6]:
        refused(call, "null")
    p = pages(table=None, refs=None)
    if K.lib().knj_synchronize() != K.KNJ_OK:  # (no GPU: the next check is the device's)
        refused(lambda: K.pages_copy(p, p, A, A, 1), "not open", K.KNJ_E_STATE)
        refused(lambda: K.pages_compact(pages(refs=None), A, A, 1), "not open", K.KNJ_E_STATE)


@pytest.mark.parametrize("kw,match", [
    (dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(type_id=K.TYPE_Q4_K), "activations"), (dict(k=None), "null"),
    (dict(v=None), "null"), (dict(n_rows=-1), "row count"), (dict(row_stride=508), "stride"), (dict(row_stride=514), "16-byte"),
    (dict(type_id=F16, row_stride=516), "16-byte"), (dict(k=A + 4), "16-byte"), (dict(n_rows=2 ** 25), "too many")])
def test_row_refusals(kw, match):
    a = dict(pages=pages(), layer=1, type_id=F32, k=A, v=A, n_rows=1, row_stride=512)
    refused(lambda: K.pages_load(**{**a, **kw}), match)
    refused(lambda: K.pages_store(start=A, **{**a, **kw}), match)


def test_array_refusals():
    p, ws = pages(), Workspace(2 ** 30)
    ws.ptr = A
    lib = K.lib()
    reserve = [None, A, A, A, A, 2 ** 30]
    for i in (1, 2, 3):
        bad = list(reserve)
        bad[i] = None
        refused(lambda: K.check(lib.knj_pages_reserve(p.ref, *bad, None)), "null")
    for i in (0, 1, 2, 3):
        bad = list(reserve)
        bad[i] = A + 2
        refused(lambda: K.check(lib.knj_pages_reserve(p.ref, *bad, None)), "aligned")
    need = K.pages_workspace(p)
    for ptr, n in ((None, need), (A, need - 1), (A + 2, need)):
        refused(lambda: K.check(lib.knj_pages_reserve(p.ref, None, A, A, A, ptr, n, None)), f"workspace of {need}")
        refused(lambda: K.check(lib.knj_pages_fork(p.ref, A, None, ptr, n, None)), f"workspace of {need}")
    refused(lambda: K.check(lib.knj_pages_fork(p.ref, None, None, A, need, None)), "null")
    refused(lambda: K.check(lib.knj_pages_fork(p.ref, A + 1, None, A, need, None)), "aligned")
    refused(lambda: K.check(lib.knj_pages_fork(p.ref, A, A + 1, A, need, None)), "aligned")
    refused(lambda: K.pages_free(p, None), "null")
    refused(lambda: K.pages_free(p, A + 2), "aligned")
    for kw, match in ((dict(start=None), "null"), (dict(rows=None), "null"), (dict(start=A + 1), "aligned"), (dict(rows=A + 2), "aligned"),
                      (dict(counts=A + 3), "aligned"), (dict(n_rows=-1), "n_rows"), (dict(n_rows=2 ** 31 - 1), "n_rows")):
        refused(lambda: K.pages_compact(p, **{**dict(start=A, rows=A, n_rows=4), **kw}), match)
    refused(lambda: K.pages_store(p, 0, F32, A, A, None, 1), "null start")
    refused(lambda: K.pages_store(p, 0, F32, A, A, A + 2, 1), "start")
    refused(lambda: K.pages_store(p, 0, F32, A, A, A, 1, counts=A + 2), "counts")
    refused(lambda: K.pages_load(p, 0, F32, A, A, 1, slots=A + 2), "slots")
    for kw, match in ((dict(dst=None), "null"), (dict(src=None), "null"), (dict(dst=A + 2), "aligned"), (dict(src=A + 1), "aligned"),
                      (dict(n=-1), "n must"), (dict(n=2 ** 24), "n must")):
        refused(lambda: K.pages_copy(p, p, **{**dict(dst=A, src=A, n=1), **kw}), match)
    for kw in (dict(n_layer=3), dict(page_size=64), dict(n_head_kv=2), dict(head_dim=64)):
        refused(lambda: K.pages_copy(p, pages(**kw), A, A, 1), "same")
    assert lib.knj_pages_free(None, A, None) == K.KNJ_E_ARG


@pytest.mark.parametrize("kw,match", [
    (dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(type_id=12), "activations"), (dict(q=None), "null"),
    (dict(out=None), "null"), (dict(prefix=None), "null"), (dict(n_rows=-1), "n_rows"), (dict(n_rows=1025, max_prefix=0), "n_rows"),
    (dict(n_head=30), "multiple"), (dict(n_head=0), "multiple"), (dict(max_prefix=-1), "n_ctx"), (dict(max_prefix=128), "n_ctx"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(q_stride=4095), "stride"), (dict(out_stride=4097), "16-byte"),
    (dict(q=A + 8), "16-byte"), (dict(prefix=A + 2), "aligned"), (dict(counts=A + 1), "aligned"), (dict(mask=A + 4), "aligned"),
    (dict(out=A, q_stride=5120), "in place")])
def test_attention_refusals(kw, match):
    a = dict(pages=pages(), layer=1, type_id=F32, q=A, out=2 * A, n_head=32, n_rows=1, prefix=A, max_prefix=100)
    refused(lambda: K.attention_pages(**{**a, **kw}), match)


def test_attention_workspace():
    p = pages(n_table=200)
    need = K.attention_pages_workspace(p, 32, 1, 6000)
    assert 0 < need <= 262144 * 132
    refused(lambda: K.attention_pages(p, 0, F32, A, 2 * A, 32, 1, A, 6000), "workspace")
    assert K.attention_pages_workspace(p, 32, 0, 10) == 0 and K.attention_pages_workspace(p, 32, 1, 6400) == 0
    most = pages(n_table=(2 ** 31 - 257) // 32, n_seq=1, n_head_kv=1)
    slots = most.desc.n_table * 32
    assert 0 < K.attention_pages_workspace(most, 8, 1000, slots - 1000) <= 262144 * 132
    assert K.attention_pages_workspace(most, 8, 1000, slots - 999) == 0
