"""GPU: the 4-bit cache in pages -- rows stored and read back, attention, pages reserved, shared, given back, moved
together and copied -- against numpy (pages_model) and float64, at the sizes and contents where they can go wrong,
and together as they are used."""
import ctypes as C

import numpy as np
import pytest

import kanjoos_amd as K
from pages_model import Pool, groups, half, values
from test_gpu_spec import (BF16, F16, F32, TYPES, close, decode, encode, hip, i32, mask_words, np_type, put,  # noqa: F401
                           streams, tree64, tree_bits)

pytestmark = pytest.mark.gpu


def upload(pool):
    """The pool on the device."""
    return K.KvPages(pool.n_layer, pool.n_page, pool.page, pool.nk, pool.D, pool.n_seq, pool.n_table, put(pool.data),
                     put(pool.table), put(pool.refs))


def same(p, pool, what=""):
    """The device's pool is the model's, byte for byte."""
    assert np.array_equal(p.table.download(np.int32).reshape(pool.table.shape), pool.table), what
    assert np.array_equal(p.refs.download(np.int32), pool.refs), what
    assert np.array_equal(p.data.download(np.uint8).reshape(pool.data.shape), pool.data), what


def own_pages(pool, rng, lengths):
    """Every sequence pages of its own for its slots, all over the pool."""
    need = [-(-int(n) // pool.page) for n in lengths]
    ids = rng.permutation(pool.n_page)[:sum(need)]
    assert len(ids) == sum(need)
    at = 0
    for s, n in enumerate(need):
        pool.table[s, :n] = ids[at:at + n]
        pool.refs[ids[at:at + n]] += 1
        at += n


# ------------------------------------------------------------------ rows

def contents(rng, shape):
    """Rows with groups of every kind: ordinary, far from zero, of no range, ranges at f16's least, ties, zeros."""
    x = rng.normal(size=shape) * np.exp(2 * rng.normal(size=shape[:-1]))[..., None] + 3 * rng.normal(size=shape[-1])
    flat = x.reshape(-1, 32)
    kind = rng.integers(0, 12, len(flat))
    flat[kind == 0] = rng.normal(size=(int((kind == 0).sum()), 1)) * 100
    flat[kind == 1] *= 2.0 ** -22
    flat[kind == 2] = 1000 + flat[kind == 2] * 1e-2
    n = int((kind == 3).sum())
    flat[kind == 3] = rng.integers(0, 31, (n, 32)) / 2 * 2.0 ** rng.integers(-20, 8, (n, 1))  # halves of a step
    flat[kind == 3, 0] = 0
    flat[kind == 3, 1] = flat[kind == 3].max(-1)
    flat[kind == 4] = 0
    flat[kind == 5] = rng.uniform(-65504, 65504, (int((kind == 5).sum()), 32))
    return x


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D,nk,n_seq,rows,page,pad", [
    (128, 4, 1, 1, 64, 0), (128, 4, 32, 1, 16, 8), (128, 1, 3, 37, 16, 0), (64, 8, 2, 50, 32, 64), (64, 3, 5, 7, 256, 0),
    (128, 5, 2, 130, 128, 16), (64, 1, 1, 9, 16, 0)])
def test_store_load(device, t, D, nk, n_seq, rows, page, pad):
    print(f"rows type {t} D {D} nk {nk} n_seq {n_seq} rows {rows} page {page} pad {pad}", flush=True)
    rng = np.random.default_rng([t, D, nk, n_seq, rows, page])
    n_table = -(-(rows + 40) // page)
    pool = Pool(rng, 3, n_seq * n_table + 2, page, nk, D, n_seq, n_table)
    own_pages(pool, rng, [n_table * page] * n_seq)
    pool.table[0, -1] = pool.n_page  # no page, in three spellings over the sequences
    pool.table[-1, 0] = [-1, -2 ** 31, 2 ** 31 - 1][n_seq % 3]
    p = upload(pool)
    stride = 2 * nk * D + pad
    raw = encode(np.concatenate([contents(rng, (n_seq * rows, 2 * nk, D)).reshape(n_seq * rows, -1),
                                 np.zeros((n_seq * rows, pad))], 1), t)
    x = decode(raw, t)[:, :2 * nk * D].reshape(n_seq, rows, 2, nk, D)
    start = rng.integers(0, 41, n_seq)
    start[0] = n_table * page - rows // 2  # the last rows fall outside
    if n_seq > 1:
        start[1] = -(rows // 2)
    counts = np.array([rows if s == 0 else max(0, rows - s) for s in range(n_seq)])
    dx = put(raw)
    size = raw.itemsize
    K.pages_store(p, 1, t, dx.ptr, dx.ptr + nk * D * size, i32(start), rows, counts=i32(counts), row_stride=stride)
    for s in range(n_seq):
        for r in range(counts[s]):
            pool.put(1, s, start[s] + r, x[s, r, 0], x[s, r, 1])
    same(p, pool)
    # read back: slots of every sequence in any order, some twice, some outside
    slots = rng.integers(-3, n_table * page + 3, (n_seq, rows)).astype(np.int32)
    for given in (slots, None):
        marks = [np.full((n_seq * rows, nk * D + 8), 7, np_type(t)) for _ in range(2)]
        out = [put(m) for m in marks]
        K.pages_load(p, 1, t, out[0], out[1], rows, slots=None if given is None else i32(given), row_stride=nk * D + 8)
        want = [m.reshape(n_seq, rows, -1).copy() for m in marks]
        all_rows = [pool.rows(1, s, n_table * page) for s in range(n_seq)]
        for s in range(n_seq):
            for r in range(rows):
                slot = r if given is None else int(given[s, r])
                if pool.where(s, slot):
                    for i in range(2):
                        with np.errstate(invalid="ignore"):
                            want[i][s, r, :nk * D] = encode(all_rows[s][i][:, slot].reshape(-1), t)
        for i in range(2):
            got = out[i].download(np_type(t), marks[i].size).reshape(want[i].shape)
            a, b = decode(got[..., :nk * D], t), decode(want[i][..., :nk * D], t)
            assert np.array_equal(a, b, equal_nan=True)
            assert np.array_equal(got[..., nk * D:], want[i][..., nk * D:])


def test_store_not_held(device):
    """Groups with infinities, NaN and magnitudes above 65504 read back as NaN, their neighbours as they are."""
    rng = np.random.default_rng(3)
    pool = Pool(rng, 1, 4, 16, 2, 64, 1, 1)
    own_pages(pool, rng, [16])
    p = upload(pool)
    x = rng.normal(size=(16, 2, 64)).astype(np.float32)
    x[0, 0, 3], x[1, 1, 40], x[2, 0, 0], x[3, 0, 63], x[4, 1, 31] = np.inf, -np.inf, np.nan, 65504.01, -1e30
    x[5, 0, :32], x[6, 0] = np.nan, np.inf
    x[7, 0, 5] = 65504
    dx = put(x)
    K.pages_store(p, 0, F32, dx, dx, i32([0]), 16)
    out = [K.DeviceBuffer(x.nbytes) for _ in range(2)]
    K.pages_load(p, 0, F32, out[0], out[1], 16)
    with np.errstate(invalid="ignore"):
        want = values(*groups(x.astype(np.float64)))
    assert np.isnan(want).any(-1).sum() == 7
    for o in out:
        assert np.array_equal(o.download(np.float32).reshape(x.shape), want.astype(np.float32), equal_nan=True)


# ------------------------------------------------------------------ attention

def filled(rng, lengths, page, nk, D, spare=3, n_layer=2, extra=2, spread=0.5):
    """A pool whose layer 1 holds random rows in every slot of every sequence's pages (the rest holds anything)."""
    n = len(lengths)
    n_table = -(-max(max(lengths), 1) // page) + extra
    pool = Pool(rng, n_layer, sum(-(-int(m) // page) for m in lengths) + spare, page, nk, D, n, n_table)
    own_pages(pool, rng, lengths)
    from pages_model import row_bytes
    x = rng.normal(size=(2, pool.n_page, nk, page, D)) * np.exp(spread * rng.normal(size=(2, pool.n_page, nk, page)))[..., None]
    held = np.unique(pool.table[pool.table >= 0])
    b = pool.blocks()
    for i in range(2):
        c, m = row_bytes(x[i][held])
        b[i][1, held], b[2 + i][1, held] = c, m
    return pool


def attend(p, t, q, T, prefix, counts, sees, nh, max_prefix=None, shared=False, scale=None, pad=0, in_place=False, layer=1,
           stream=None):
    """attention_pages on host arrays; rows of q and out `pad` elements apart."""
    n, D = p.desc.n_seq, p.desc.head_dim
    width = nh * D
    rows = np.full((n * T, width + pad), 7.0)
    mark = encode(rows, t)
    rows[:, :width] = q.reshape(n * T, width)
    dq = put(encode(rows, t))
    out = dq if in_place else put(mark)
    max_prefix = int(max(prefix)) if max_prefix is None else max_prefix
    ws = K.DeviceBuffer(K.attention_pages_workspace(p, nh, T, max_prefix) + 64)
    ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))  # NaN wherever nothing is written
    K.attention_pages(p, layer, t, dq, out, nh, T, i32(prefix), max_prefix, ws, counts=None if counts is None else i32(counts),
                      mask=None if sees is None else put(mask_words(sees)), mask_shared=shared, scale=scale,
                      q_stride=width + pad, out_stride=width + pad)
    got = out.download(np_type(t), mark.size).reshape(n * T, -1)
    base = encode(rows, t) if in_place else mark
    assert np.array_equal(got[:, width:], base[:, width:])
    return decode(got[:, :width], t).reshape(n, T, nh, D), decode(base[:, :width], t).reshape(n, T, nh, D)


def caches(pool, n, layer=1):
    """Keys and values [n_seq][nk][n][D] of the first n slots (zeros where a sequence has fewer pages)."""
    out = [np.zeros((pool.n_seq, pool.nk, n, pool.D)) for _ in range(2)]
    for s in range(pool.n_seq):
        for i, x in enumerate(pool.rows(layer, s, min(n, pool.n_table * pool.page))):
            out[i][s, :, :x.shape[1]] = x
    return out


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D,nh,nk,T,page,prefixes", [
    (128, 32, 4, 1, 64, (0, 1, 31, 32, 63)), (128, 8, 1, 2, 16, (64, 65, 126, 127, 128, 129)), (128, 12, 4, 5, 32, (0, 3, 200, 383)),
    (128, 4, 4, 16, 256, (1, 500)), (64, 14, 2, 9, 16, (0, 64, 130)), (64, 16, 2, 3, 128, (1000, 7)), (128, 10, 2, 13, 64, (250, 64)),
    (64, 8, 8, 66, 32, (70, 0)), (128, 24, 1, 7, 64, (129, 300)), (128, 32, 4, 25, 16, (190,)), (128, 32, 4, 1, 64, (2100, 900, 15)),
    (64, 16, 2, 1, 16, (1500,)), (128, 8, 8, 1, 32, (40, 0, 700))])
def test_attention(device, t, D, nh, nk, T, page, prefixes):
    """Trees over prefixes on both sides of the tiles' and the pages' borders, groups that are no power of two,
    sequences of different lengths."""
    print(f"attention type {t} D {D} heads {nh}/{nk} T {T} page {page} prefixes {prefixes}", flush=True)
    rng = np.random.default_rng([D, nh, nk, T, page, t])
    n = len(prefixes)
    pool = filled(rng, [m + T for m in prefixes], page, nk, D)
    p = upload(pool)
    kv = caches(pool, max(prefixes) + T)
    sees = np.stack([tree_bits(rng, T) for _ in range(n)])
    counts = np.array([max(1, T - s % 3) for s in range(n)])
    q = decode(encode(1.5 * rng.normal(size=(n, T, nh, D)), t), t)
    got, before = attend(p, t, q, T, prefixes, counts, sees, nh, pad=16)
    want, bound = tree64(q, kv, prefixes, counts, sees, D ** -0.5, t)
    for s in range(n):
        close(got[s, :counts[s]], want[s, :counts[s]], bound[s, :counts[s]], f"prefix {prefixes[s]}")
        assert np.array_equal(got[s, counts[s]:], before[s, counts[s]:])  # rows past the drafts
    again, _ = attend(p, t, q, T, prefixes, counts, sees, nh, pad=16, in_place=True)
    for s in range(n):
        assert np.array_equal(again[s, :counts[s]], got[s, :counts[s]])
    same(p, pool)


@pytest.mark.parametrize("T,nh", [(1, 6), (40, 6), (64, 2), (65, 6), (130, 2)])
@pytest.mark.parametrize("page", [16, 128])
def test_attention_chain(device, T, nh, page):
    """No mask: row t sees rows 0..t, the same bits as with that mask, its own a sequence or one shared; a looser bound
    on the prefixes changes the split alone."""
    rng = np.random.default_rng([T, page])
    nk, D, prefixes = 2, 128, [0, 77]
    pool = filled(rng, [T, 77 + T], page, nk, D, extra=3000 // page + 1)
    p = upload(pool)
    kv = caches(pool, 77 + T)
    q = rng.normal(size=(2, T, nh, D)).astype(np.float32).astype(np.float64)
    sees = np.stack([np.tril(np.ones((T, T), bool))] * 2)
    got, _ = attend(p, F32, q, T, prefixes, None, None, nh)
    want, bound = tree64(q, kv, prefixes, [T, T], sees, D ** -0.5, F32)
    close(got, want, bound, "chain")
    assert np.array_equal(attend(p, F32, q, T, prefixes, None, sees, nh)[0], got)
    assert np.array_equal(attend(p, F32, q, T, prefixes, None, sees[:1], nh, shared=True)[0], got)
    got, _ = attend(p, F32, q, T, prefixes, None, None, nh, max_prefix=3000 - T)
    close(got, want, bound, "loose bound")


def test_attention_lengths_held(device):
    """Prefixes and counts outside their range are held to it."""
    rng = np.random.default_rng(1)
    nh, nk, D, T = 4, 2, 64, 3
    pool = filled(rng, [96] * 5, 16, nk, D, extra=0)
    p = upload(pool)
    kv = caches(pool, 96)
    q = rng.normal(size=(5, T, nh, D)).astype(np.float32).astype(np.float64)
    sees = np.stack([tree_bits(rng, T) for _ in range(5)])
    got, before = attend(p, F32, q, T, [-7, 5000, 2 ** 31 - 1, 20, -2 ** 31], [T, 2 ** 31 - 1, T, -1, 0], sees, nh, max_prefix=90)
    held, counts = [0, 90, 90, 20, 0], [T, T, T, 0, 0]
    want, bound = tree64(q, kv, held, counts, sees, D ** -0.5, F32)
    for s in range(5):
        close(got[s, :counts[s]], want[s, :counts[s]], bound[s, :counts[s]], f"sequence {s}")
        assert np.array_equal(got[s, counts[s]:], before[s, counts[s]:])


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("T,nh", [(1, 2), (6, 2), (6, 8), (20, 4), (40, 8), (40, 16)])
def test_attention_unseen_slots(device, t, T, nh):
    """Slots that a row does not see count for nothing, whatever they hold: NaN and huge values in unseen rows and past
    them; a row that sees nothing gives zeros; one that sees a spoilt value gives NaN."""
    print(f"unseen type {t} T {T} heads {nh}", flush=True)
    rng = np.random.default_rng([t, T])
    nk, D, prefixes = 2, 64, np.array([0, 61, 128])
    pool = filled(rng, [200] * 3, 32, nk, D)
    # every byte past the rows set: NaN in step and lowest value
    for s in range(3):
        for slot in range(prefixes[s] + T, 200):
            at = pool.where(s, slot)
            for b in pool.blocks():
                b[1, at[0], :, at[1]] = 0xFF
    for s in range(3):
        for r in range(min(T, 5)):
            x = rng.normal(size=(2, nk, D)) * [1, 1e4, 1, 1, 1e-3][r]
            if r == 2:
                x[1, :, 5], x[0, :, 7] = np.inf, -np.inf
            if r == 3:
                x[:, :, 0] = np.nan
            pool.put(1, s, prefixes[s] + r, *x)
    p = upload(pool)
    kv = caches(pool, 128 + T)
    sees = np.zeros((3, T, T), bool)
    for i in range(T):
        sees[:, i, i] = i not in (1, 2, 3)
        sees[:, i, 0] = True
    sees[:, 0] = False  # nothing but the prefix: nothing at all with a prefix of 0
    if T > 5:
        sees[:, 5, 4] = True
        sees[0, 2, 2] = sees[1, 2, 3] = True  # a spoilt value seen
    q = decode(encode(rng.normal(size=(3, T, nh, D)), t), t)
    got, _ = attend(p, t, q, T, prefixes, None, sees, nh)
    with np.errstate(invalid="ignore", over="ignore"):
        want, bound = tree64(q, kv, prefixes, [T] * 3, sees, D ** -0.5, t)
    assert np.all(want[0, 0] == 0)
    # (a spoilt group is 32 of a row's dims, and a row that sees one is NaN in all)
    close(got, want, bound, "unseen")
    assert np.all(got[0, 0] == 0)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D,T,nh,nk,page,prefixes,limit", [
    (128, 1, 16, 2, 64, (101, 128, 135, 129), None), (64, 2, 16, 2, 16, (1000, 111, 130, 160), None),  # up to 16 columns
    (128, 3, 32, 4, 32, (101, 128, 131, 130) * 4, None), (64, 17, 2, 2, 64, (101, 200), 32000),  # 17 to 32
    (64, 9, 16, 2, 64, (101, 128, 131, 200), None), (128, 20, 6, 2, 16, (101, 160), None),  # more
    (128, 66, 4, 2, 64, (101, 192, 163, 161), 32000), (128, 130, 2, 1, 128, (129, 101, 190), 32000)])  # many, work enough
def test_attention_prefix_value_not_held(device, t, D, T, nh, nk, page, prefixes, limit):
    """One value group of a prefix slot that is not held, the last slot's or the hundredth before the drafts: NaN in
    that group's dims of every row of its kv head, whichever tile the slot falls into, and nowhere else."""
    print(f"prefix value not held: type {t} D {D} T {T} heads {nh}/{nk} prefixes {prefixes}", flush=True)
    rng = np.random.default_rng([D, T, nh, t])
    n = len(prefixes)
    pool = filled(rng, [m + T for m in prefixes], page, nk, D, extra=0 if limit is None else (limit + T) // page + 1)
    clean = caches(pool, max(prefixes) + T)
    spoilt = np.zeros((n, nk, D), bool)
    for s, P in enumerate(prefixes):
        slot, h, g = P - 1 if s % 2 == 0 else P - 100, s % nk, (s // 2) % (D // 32)
        at = pool.where(s, slot)
        pool.blocks()[3][1, at[0], h, at[1]].view(np.uint32)[g] = 0x7E000000
        spoilt[s, h, 32 * g:32 * g + 32] = True
    p = upload(pool)
    kv = caches(pool, max(prefixes) + T)
    q = decode(encode(rng.normal(size=(n, T, nh, D)), t), t)
    for chain in (True, False):
        sees = np.stack([np.tril(np.ones((T, T), bool)) if chain else tree_bits(rng, T) for _ in range(n)])
        got, _ = attend(p, t, q, T, prefixes, None, None if chain else sees, nh, max_prefix=limit)
        want, bound = tree64(q, kv, prefixes, [T] * n, sees, D ** -0.5, t)
        without, off = tree64(q, clean, prefixes, [T] * n, sees, D ** -0.5, t)
        by_head = np.repeat(spoilt, nh // nk, 1)[:, None]
        assert np.array_equal(np.isnan(want), np.broadcast_to(by_head, want.shape))
        close(got, want, bound, "spoilt")
        close(np.where(by_head, 0.0, got), np.where(by_head, 0.0, without), off, "the rest")


@pytest.mark.parametrize("T,nh", [(1, 8), (3, 8), (20, 8)])
def test_attention_without_a_page(device, T, nh):
    """Slots whose page is outside the pool hold NaN: sequences that reach one are NaN, others and rows past the slots
    are not touched by it; nothing outside the pool is read."""
    rng = np.random.default_rng(T)
    nk, D, prefixes = 2, 128, [100, 40, 300, 0]
    pool = filled(rng, [m + T for m in prefixes], 16, nk, D)
    pool.table[0, 3] = pool.n_page
    pool.table[2, 0] = -5
    pool.table[1, 5:] = 2 ** 31 - 1  # behind the sequence's slots
    pool.table[3, 2:] = -2 ** 31
    p = upload(pool)
    kv = caches(pool, 300 + T)
    q = rng.normal(size=(4, T, nh, D)).astype(np.float32).astype(np.float64)
    sees = np.stack([tree_bits(rng, T) for _ in range(4)])
    got, _ = attend(p, F32, q, T, prefixes, None, sees, nh)
    assert np.isnan(got[0]).all() and np.isnan(got[2]).all()
    for s in (1, 3):
        want, bound = tree64(q[s:s + 1], [x[s:s + 1] for x in kv], [prefixes[s]], [T], sees[s:s + 1], D ** -0.5, F32)
        close(got[s], want[0], bound[0], f"sequence {s}")


@pytest.mark.parametrize("size", [1e-30, 1e-4, 1.0, 3e4, 1e9])
@pytest.mark.parametrize("T", [1, 4])
def test_attention_magnitudes(device, size, T):
    """Queries of any size whose scores stay ordinary: the scale takes the size out again where it may."""
    rng = np.random.default_rng(7)
    nh, nk, D = 8, 2, 128
    pool = filled(rng, [300], 64, nk, D)
    p = upload(pool)
    kv = caches(pool, 300)
    scale = float(np.float32(min(1e6, max(1e-6, D ** -0.5 / size))))
    q = (rng.normal(size=(1, T, nh, D)) * size).astype(np.float32).astype(np.float64)
    sees = np.stack([tree_bits(rng, T)])
    got, _ = attend(p, F32, q, T, [300 - T], None, sees, nh, scale=scale)
    want, bound = tree64(q, kv, [300 - T], [T], sees, scale, F32)
    close(got, want, bound, f"size {size}")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,nh,rising", [(1, 4, True), (1, 4, False), (8, 8, True), (30, 8, True), (70, 8, True)])
def test_attention_drifting(device, t, T, nh, rising):
    """Scores that rise or fall along the slots by far more than f16 or an exponent's reference holds."""
    rng = np.random.default_rng([t, T])
    nk, D, P = 1, 64, 1500
    pool = filled(rng, [P + T], 64, nk, D)
    d = rng.normal(size=D)
    drift = np.linspace(-40, 40, P + T) * (1 if rising else -1)
    rows = np.stack([drift[:, None] * d / (d @ d) * 8 + rng.normal(size=(P + T, D)) * 0.3, rng.normal(size=(P + T, D))])
    for slot in range(P + T):
        pool.put(1, 0, slot, rows[0][slot][None], rows[1][slot][None])
    p = upload(pool)
    kv = caches(pool, P + T)
    q = decode(encode(np.broadcast_to(4 * d, (1, T, nh, D)) + 0.1 * rng.normal(size=(1, T, nh, D)), t), t)
    sees = np.stack([tree_bits(rng, T)])
    got, _ = attend(p, t, q, T, [P], None, sees, nh)
    want, bound = tree64(q, kv, [P], [T], sees, D ** -0.5, t)
    close(got, want, bound, "drift")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D,T,nh,nk,P", [(128, 64, 32, 4, 260), (128, 200, 8, 1, 1100), (64, 96, 16, 2, 700), (128, 33, 16, 8, 90),
                                         (128, 1024, 4, 2, 5)])
def test_attention_wide(device, t, D, T, nh, nk, P):
    """Many columns: every tile's shape, and pieces of prompts.  Rows at both ends and a sample are compared."""
    rng = np.random.default_rng([t, D, T, nh])
    pool = filled(rng, [P + T], 64, nk, D)
    p = upload(pool)
    kv = caches(pool, P + T)
    q = decode(encode(rng.normal(size=(1, T, nh, D)), t), t)
    got, _ = attend(p, t, q, T, [P], None, None, nh)
    pick = np.unique(np.concatenate([[0, 1, T - 2, T - 1], rng.integers(0, T, 20)]))
    sees = np.tril(np.ones((T, T), bool))
    for i in pick:
        want, bound = tree64(q[:, i:i + 1], kv, [P + i], [1], sees[None, :1, :1], D ** -0.5, t)
        close(got[:, i:i + 1], want, bound, f"row {i}")


# A loose bound on the prefixes asks for many columns' kernel over short sequences too.
LOOSE = 32000


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,nh,nk,page,prefixes,D", [
    (66, 8, 4, 16, (0, 1, 61, 62, 63, 64, 126, 127, 500), 128), (25, 32, 2, 64, (190, 3, 64), 128),
    (130, 5, 1, 32, (0, 127, 128, 700), 128), (17, 4, 1, 256, (100, 257, 0, 40, 1900), 128), (257, 3, 3, 128, (5, 255), 128),
    (25, 4, 2, 32, (0, 64, 500, 63), 128), (44, 8, 2, 16, (0, 127, 300), 64), (20, 6, 2, 64, (1, 64, 130, 0), 64)])
def test_attention_many_columns(device, t, T, nh, nk, page, prefixes, D):
    """Trees with what not every row sees: NaN and huge values in unseen rows and past them, rows that see nothing,
    rows that see a spoilt value; sequences with fewer rows, one of them with none."""
    print(f"many columns type {t} D {D} T {T} heads {nh}/{nk} page {page} prefixes {prefixes}", flush=True)
    rng = np.random.default_rng([T, nh, page, t])
    n = len(prefixes)
    pool = filled(rng, [m + T + 20 for m in prefixes], page, nk, D, extra=(LOOSE + T) // page + 1)
    counts = np.array([T if s == 0 else max(T - 40 * s, 0) for s in range(n)])
    sees = np.stack([tree_bits(rng, T) for _ in range(n)])
    sees[:, :, 2:5] = False
    sees[:, 0] = False
    for s, P in enumerate(prefixes):
        for slot in range(P + counts[s], P + T + 20):  # every byte past the rows set: NaN in step and lowest value
            at = pool.where(s, slot)
            for b in pool.blocks():
                b[1, at[0], :, at[1]] = 0xFF
        x = rng.normal(size=(3, 2, nk, D))
        x[0, 1, :, 5], x[0, 0, :, 7] = np.inf, -np.inf
        x[1, :, :, D - 28] = np.nan
        x[2] *= 1e4
        for r in range(min(3, counts[s] - 2)):
            pool.put(1, s, P + 2 + r, *x[r])
    sees[1 % n, 6, 2] = sees[0, 9, 3] = True  # a spoilt value seen
    p = upload(pool)
    kv = caches(pool, max(prefixes) + T)
    q = decode(encode(1.5 * rng.normal(size=(n, T, nh, D)), t), t)
    got, before = attend(p, t, q, T, prefixes, counts, sees, nh, pad=16, max_prefix=LOOSE)
    with np.errstate(invalid="ignore", over="ignore"):
        want, bound = tree64(q, kv, prefixes, counts, sees, D ** -0.5, t)
    for s in range(n):
        close(got[s, :counts[s]], want[s, :counts[s]], bound[s, :counts[s]], f"prefix {prefixes[s]}")
        assert np.array_equal(got[s, counts[s]:], before[s, counts[s]:])  # rows past the drafts
        if prefixes[s] == 0 and counts[s]:
            assert np.all(got[s, 0] == 0)
    again, _ = attend(p, t, q, T, prefixes, counts, sees, nh, pad=16, max_prefix=LOOSE, in_place=True)
    for s in range(n):
        assert np.array_equal(again[s, :counts[s]], got[s, :counts[s]], equal_nan=True)
    same(p, pool)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("T,nh,prefixes,loose", [(65, 6, (0, 77), True), (130, 2, (64, 1), True), (350, 12, (0, 41), False),
                                                 (700, 8, (0,), False)])
def test_attention_many_columns_chain(device, t, T, nh, prefixes, loose):
    """No mask: row t sees rows 0..t, the same bits as with that mask, its own a sequence or one shared; a spoilt value
    makes NaN of the rows from its own on, alike with a mask and without."""
    print(f"many columns, chain: type {t} T {T} heads {nh} prefixes {prefixes}", flush=True)
    rng = np.random.default_rng([T, nh, t])
    nk, D, n = 1, 128, len(prefixes)
    pool = filled(rng, [m + T for m in prefixes], 32, nk, D, extra=(LOOSE + T) // 32 + 1)
    x = rng.normal(size=(2, nk, D))
    x[1, :, 40] = np.inf
    pool.put(1, n - 1, prefixes[-1] + T - 30, *x)
    p = upload(pool)
    kv = caches(pool, max(prefixes) + T)
    q = decode(encode(rng.normal(size=(n, T, nh, D)), t), t)
    sees = np.stack([np.tril(np.ones((T, T), bool))] * n)
    limit = LOOSE if loose else None
    got, _ = attend(p, t, q, T, prefixes, None, None, nh, max_prefix=limit)
    with np.errstate(invalid="ignore"):
        want, bound = tree64(q, kv, prefixes, [T] * n, sees, D ** -0.5, t)
    close(got, want, bound, "chain")
    assert np.isnan(got[n - 1, T - 30:]).all()
    assert np.array_equal(attend(p, t, q, T, prefixes, None, sees, nh, max_prefix=limit)[0], got, equal_nan=True)
    assert np.array_equal(attend(p, t, q, T, prefixes, None, sees[:1], nh, shared=True, max_prefix=limit)[0], got, equal_nan=True)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,nh,nk,page,prefixes", [
    (20, 32, 4, 16, tuple(range(33))), (16, 48, 4, 32, (0, 1, 15, 17, 48) * 8), (40, 16, 4, 16, (0, 30, 60, 88) * 14),  # no merge
    (70, 32, 1, 64, (0, 61)), (17, 128, 1, 16, (0,)), (260, 8, 1, 32, (30,))])  # more than 2048 columns
def test_attention_many_columns_short(device, t, T, nh, nk, page, prefixes):
    """Many columns over few slots, of many sequences (no split to merge) or of one (more columns than an XCD holds at
    once): trees and chains, sequences with fewer rows; a sample of the rows is compared."""
    print(f"many columns, short: type {t} T {T} heads {nh}/{nk} prefixes {len(prefixes)}", flush=True)
    rng = np.random.default_rng([T, nh, page, t])
    n, D = len(prefixes), 128
    pool = filled(rng, [m + T for m in prefixes], page, nk, D)
    p = upload(pool)
    kv = caches(pool, max(prefixes) + T)
    counts = np.array([T if s % 3 == 0 else max(T - s, 0) for s in range(n)])
    q = decode(encode(1.5 * rng.normal(size=(n, T, nh, D)), t), t)
    trees = np.stack([tree_bits(rng, T) for _ in range(n)])
    trees[:, 1] = False  # the prefix alone
    below = np.tril(np.ones((T, T), bool))
    for sees, mask in ((trees, trees), (np.stack([below] * n), None)):
        got, before = attend(p, t, q, T, prefixes, counts, mask, nh, pad=16)
        for s in range(n):
            assert np.array_equal(got[s, counts[s]:], before[s, counts[s]:])  # rows past the drafts
            h = np.unique(rng.integers(0, nh, 4))  # (heads one by one: each has its kv head's cache)
            for x in h if counts[s] else []:
                one = [c[s:s + 1, x * nk // nh:x * nk // nh + 1] for c in kv]
                want, bound = tree64(q[s:s + 1, :, x:x + 1], one, [prefixes[s]], [counts[s]], sees[s:s + 1], D ** -0.5, t)
                close(got[s:s + 1, :counts[s], x:x + 1], want[:, :counts[s]], bound[:, :counts[s]], f"sequence {s} head {x}")
    assert np.array_equal(attend(p, t, q, T, prefixes, counts, below[None], nh, shared=True, pad=16)[0], got)
    again, _ = attend(p, t, q, T, prefixes, counts, None, nh, pad=16, in_place=True)
    for s in range(n):
        assert np.array_equal(again[s, :counts[s]], got[s, :counts[s]])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rising", [True, False])
def test_attention_many_columns_drifting(device, t, rising):
    """Scores that rise or fall along the slots by far more than f16 or an exponent's reference holds; a sequence
    without a page beside it."""
    rng = np.random.default_rng([t, rising])
    T, nh, nk, D, P = 70, 8, 1, 128, 1500
    pool = filled(rng, [P + T, 200 + T], 64, nk, D, extra=LOOSE // 64)
    d = rng.normal(size=D)
    drift = np.linspace(-40, 40, P + T) * (1 if rising else -1)
    rows = np.stack([drift[:, None] * d / (d @ d) * 8 + rng.normal(size=(P + T, D)) * 0.3, rng.normal(size=(P + T, D))])
    for slot in range(P + T):
        pool.put(1, 0, slot, rows[0][slot][None], rows[1][slot][None])
    pool.table[1, 2] = -7
    pool.table[0, (P + T + 63) // 64:] = 2 ** 31 - 1  # behind the sequence's slots
    p = upload(pool)
    kv = [x[:1] for x in caches(pool, P + T)]
    q = decode(encode(np.broadcast_to(4 * d, (2, T, nh, D)) + 0.1 * rng.normal(size=(2, T, nh, D)), t), t)
    sees = np.stack([tree_bits(rng, T)] * 2)
    got, _ = attend(p, t, q, T, [P, 200], None, sees, nh, max_prefix=LOOSE)
    want, bound = tree64(q[:1], kv, [P], [T], sees[:1], D ** -0.5, t)
    close(got[:1], want, bound, "drift")
    assert np.isnan(got[1]).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D,T,nh,nk,page,prefixes,loose", [
    (128, 4, 16, 2, 64, (0, 500, 31, 1900), True), (64, 17, 2, 2, 16, (64, 200), True), (128, 9, 6, 2, 32, (1, 1000), True),
    (128, 3, 32, 4, 64, tuple(range(0, 500, 31)), False), (64, 8, 24, 8, 128, (0, 1, 30, 32, 33, 450, 64, 90), False)])
def test_attention_two_column_tiles(device, t, D, T, nh, nk, page, prefixes, loose):
    """17 to 32 columns with work enough: trees with what not every row sees, rows that see nothing, rows that see a
    spoilt value, sequences with fewer rows; the same bits with a mask that sees all before it as without."""
    print(f"two tiles type {t} D {D} T {T} heads {nh}/{nk} page {page} prefixes {prefixes}", flush=True)
    rng = np.random.default_rng([T, nh, page, t])
    n = len(prefixes)
    pool = filled(rng, [m + T + 20 for m in prefixes], page, nk, D, extra=(LOOSE + T) // page + 1 if loose else 2)
    counts = np.array([T if s % 3 == 0 else max(T - s, 0) for s in range(n)])
    sees = np.stack([tree_bits(rng, T) for _ in range(n)])
    sees[:, :, 1] = False
    sees[:, 0] = False
    for s, P in enumerate(prefixes):
        for slot in range(P + counts[s], P + T + 20):  # every byte past the rows set: NaN in step and lowest value
            at = pool.where(s, slot)
            for b in pool.blocks():
                b[1, at[0], :, at[1]] = 0xFF
        x = rng.normal(size=(2, nk, D))
        x[1, :, 5], x[0, :, 7] = np.inf, -np.inf
        if counts[s] > 1:
            pool.put(1, s, P + 1, *x)
    sees[0, 2, 1] = True  # a spoilt value seen
    p = upload(pool)
    kv = caches(pool, max(prefixes) + T)
    q = decode(encode(1.5 * rng.normal(size=(n, T, nh, D)), t), t)
    limit = LOOSE if loose else None
    got, before = attend(p, t, q, T, prefixes, counts, sees, nh, pad=16, max_prefix=limit)
    with np.errstate(invalid="ignore", over="ignore"):
        want, bound = tree64(q, kv, prefixes, counts, sees, D ** -0.5, t)
    for s in range(n):
        close(got[s, :counts[s]], want[s, :counts[s]], bound[s, :counts[s]], f"prefix {prefixes[s]}")
        assert np.array_equal(got[s, counts[s]:], before[s, counts[s]:])  # rows past the drafts
        if prefixes[s] == 0 and counts[s]:
            assert np.all(got[s, 0] == 0)
    assert np.isnan(got[0, 2]).all()
    below = np.tril(np.ones((1, T, T), bool))
    chain, _ = attend(p, t, q, T, prefixes, counts, None, nh, max_prefix=limit)
    again, _ = attend(p, t, q, T, prefixes, counts, below, nh, shared=True, max_prefix=limit)
    for s in range(n):
        assert np.array_equal(again[s, :counts[s]], chain[s, :counts[s]], equal_nan=True)


@pytest.mark.parametrize("T", [1, 3])
def test_attention_long(device, T):
    """Long contexts of several splits; layers and pages beyond 2^32 bytes."""
    rng = np.random.default_rng(T)
    nk, nh, D, page, P = 2, 8, 128, 64, 33000
    n_page = 120000  # 2.4 GB a layer
    need = -(-(P + T) // page)
    d = K.KvPages.allocate(2, n_page, page, nk, D, 1, need)
    ids = n_page - 1 - np.arange(need)
    ids[::2] = np.arange(need)[::2]
    d.table.upload(ids.astype(np.int32))
    x = (rng.normal(size=(2, P + T, nk, D)) * np.exp(0.5 * rng.normal(size=(2, P + T, nk)))[..., None]).astype(np.float32)
    x[0] += 2 * rng.normal(size=D).astype(np.float32)
    bufs = [put(a) for a in x]
    K.pages_store(d, 1, F32, bufs[0], bufs[1], i32([0]), P + T)
    kv = [values(*groups(a.astype(np.float64))).transpose(1, 0, 2)[None] for a in x]
    q = rng.normal(size=(1, T, nh, D)).astype(np.float32).astype(np.float64)
    sees = np.stack([tree_bits(rng, T)])
    got, _ = attend(d, F32, q, T, [P], None, sees, nh)
    want, bound = tree64(q, kv, [P], [T], sees, D ** -0.5, F32)
    close(got, want, bound, "long")


@pytest.mark.parametrize("T", [1, 2])
def test_attention_many_sequences(device, T):
    """As many sequences as there may be, most of them short or empty; shared pages."""
    rng = np.random.default_rng(T)
    n, nk, nh, D, page = 4096, 1, 4, 64, 16
    prefixes = rng.integers(0, 40, n)
    pool = filled(rng, [48] * 50, page, nk, D)
    table = np.repeat(pool.table, 82, 0)[:n]
    pool.table, pool.n_seq = table, n
    p = upload(pool)
    kv = caches(pool, 48)
    q = rng.normal(size=(n, T, nh, D)).astype(np.float32).astype(np.float64)
    sees = np.stack([np.tril(np.ones((T, T), bool))] * n)
    counts = rng.integers(0, T + 1, n)
    got, before = attend(p, F32, q, T, prefixes, counts, None, nh)
    want, bound = tree64(q, kv, prefixes, counts, sees, D ** -0.5, F32)
    for s in range(n):
        assert np.array_equal(got[s, counts[s]:], before[s, counts[s]:])
        want[s, counts[s]:], bound[s, counts[s]:] = got[s, counts[s]:], 0
    close(got, want, bound, "many")


def test_attention_same_bits_alone(device):
    """A sequence's rows do not hang on the other sequences' contents."""
    rng = np.random.default_rng(5)
    nk, nh, D, T = 2, 8, 128, 3
    prefixes = [200, 500, 90]
    pool = filled(rng, [m + T for m in prefixes], 32, nk, D)
    p = upload(pool)
    q = rng.normal(size=(3, T, nh, D)).astype(np.float32).astype(np.float64)
    got, _ = attend(p, F32, q, T, prefixes, None, None, nh)
    spoilt = pool.table[1][pool.table[1] >= 0]
    pool.data[1, spoilt] = 0xFF
    q[1] = np.nan
    again, _ = attend(upload(pool), F32, q, T, prefixes, None, None, nh)
    assert np.array_equal(again[[0, 2]], got[[0, 2]]) and np.isnan(again[1]).all()


# ------------------------------------------------------------------ the table

def workspace(p):
    ws = K.DeviceBuffer(K.pages_workspace(p) + 16)
    ws.upload(np.full(ws.nbytes, 0xAB, np.uint8))
    return ws


def reserve(p, start, length, want):
    missing = i32([77])
    K.pages_reserve(p, i32(length), i32(want), missing, workspace(p), start=None if start is None else i32(start))
    return int(missing.download(np.int32)[0])


@pytest.mark.parametrize("D,n_seq,n_page,page,n_table,seed", [
    (64, 5, 40, 16, 12, 0), (128, 9, 70, 32, 9, 1), (64, 33, 500, 16, 20, 2), (128, 3, 9, 256, 4, 3), (64, 70, 5000, 16, 70, 4),
    (64, 1, 3000, 16, 2500, 5), (64, 1500, 9000, 16, 5, 6), (64, 300, 6000, 16, 40, 7)])
def test_table_steps(device, D, n_seq, n_page, page, n_table, seed):
    """Random steps over one pool: reserve (with and without a start, with too few pages too), fork, free, store, compact,
    against the model after each."""
    rng = np.random.default_rng(seed)
    pool = Pool(rng, 2, n_page, page, 2, D, n_seq, n_table)
    p = upload(pool)
    length = np.zeros(n_seq, np.int64)
    most = n_table * page
    for step in range(14):
        print(f"seed {seed} step {step}", flush=True)
        if step in (3, 7, 10):
            parent = rng.integers(-1, n_seq + 1, n_seq)
            if step == 7:
                parent = np.where(rng.random(n_seq) < 0.5, np.arange(n_seq), parent)
            ok = (parent >= 0) & (parent < n_seq)
            keep = np.where(ok, length[np.clip(parent, 0, n_seq - 1)], 0)
            if step == 10:
                K.pages_fork(p, i32(parent), workspace(p))
                pool.fork(parent)
            else:
                keep = np.where(rng.random(n_seq) < 0.3, keep // 2, keep)
                K.pages_fork(p, i32(parent), workspace(p), keep=i32(keep))
                pool.fork(parent, keep)
            length = keep
            same(p, pool, "fork")
        if step in (5, 9):
            keep = np.where(rng.random(n_seq) < 0.6, rng.integers(0, most + page, n_seq), -1)
            keep = np.minimum(keep, length)
            keep[rng.integers(0, n_seq)] = -2 ** 31
            K.pages_free(p, i32(keep))
            pool.free(keep)
            length = np.where(keep >= 0, keep, length)
            same(p, pool, "free")
        grow = rng.integers(0, [3, page + 3, 3 * page][step % 3], n_seq) * (rng.random(n_seq) < 0.8)
        want = np.minimum(length + grow, most + (step == 6) * 40)
        start = None if step % 2 else np.maximum(length - rng.integers(0, 2 * page, n_seq), -5)
        got = reserve(p, start, length, want)
        short = pool.reserve(length if start is None else start, length, want)
        assert got == short, (got, short)
        same(p, pool, "reserve")
        if short == 0:
            length = np.minimum(want, most)
        if step % 4 == 2:  # rows among the last ones kept, after pages of their own
            first = np.maximum(length - rng.integers(1, 40, n_seq), 0)
            short = pool.reserve(first, length, length)
            assert reserve(p, first, length, length) == short
            if short == 0:
                n_rows = 40
                rows, counts = np.zeros((n_seq, n_rows), np.int64), np.zeros(n_seq, np.int64)
                for s in range(n_seq):
                    pick = np.flatnonzero(rng.random(int(length[s] - first[s])) < 0.5)
                    counts[s] = len(pick)
                    rows[s, :len(pick)] = first[s] + pick
                K.pages_compact(p, i32(first), i32(rows), n_rows, counts=i32(counts))
                pool.compact(first, rows, counts)
                same(p, pool, "compact")
                K.pages_free(p, i32(first + counts))
                pool.free(first + counts)
                length = first + counts
                same(p, pool, "free after compact")


def test_reserve_order_and_sharing(device):
    """Lowest free pages in order of sequence and entry; of a page that all its holders write the last keeps it; a page
    that a caller holds beside the table is copied by all; nothing changes where pages are short."""
    rng = np.random.default_rng(0)
    pool = Pool(rng, 1, 12, 16, 1, 64, 4, 3)
    pool.table[0, 0] = pool.table[1, 0] = pool.table[3, 0] = 5
    pool.table[2, 0] = 7
    pool.refs[5], pool.refs[7], pool.refs[1] = 3, 2, 1
    p = upload(pool)
    length, want = [10, 10, 10, 10], [20, 11, 12, 10]
    assert reserve(p, None, length, want) == 0 == pool.reserve(length, length, want)
    # 0 copies 5 into 0 and gets 2 for its next entry, 1 copies into 3, 2's has another holder: 4
    assert pool.table[:, :2].tolist() == [[0, 2], [3, -1], [4, -1], [5, -1]] and pool.refs[5] == 1
    same(p, pool)
    want = [20, 11, 12, 11]
    assert reserve(p, None, length, want) == 0 == pool.reserve(length, length, want)
    same(p, pool, "nothing to do")
    want = [48, 48, 48, 48]
    short = reserve(p, None, length, want)
    assert short == pool.reserve(length, length, want) == 2  # seven entries, five free pages
    same(p, pool, "short")
    pool.refs[11] = 0
    pool.table[2, 0], pool.refs[4] = 5, 0
    pool.refs[5], pool.refs[7] = 2, 0
    p = upload(pool)
    assert reserve(p, None, length, [10, 10, 20, 20]) == 0 == pool.reserve(length, length, [10, 10, 20, 20])
    assert pool.table[3, 0] == 5 and pool.table[2, 0] == 4 and pool.refs[5] == 1
    same(p, pool, "the last holder keeps it")


def test_entries_that_are_none(device):
    """Entries outside the pool count nothing, whatever they are."""
    rng = np.random.default_rng(0)
    pool = Pool(rng, 1, 30, 16, 1, 64, 3, 6)
    own_pages(pool, rng, [60, 30, 96])
    pool.table[0, 2], pool.table[1, 3], pool.table[2, 0] = 30, 2 ** 31 - 1, -2 ** 31
    pool.refs[:] = np.bincount(pool.table[(pool.table >= 0) & (pool.table < 30)], minlength=30)
    p = upload(pool)
    parent, keep = [2, 0, 1], [96, 64, 2 ** 31 - 1]
    K.pages_fork(p, i32(parent), workspace(p), keep=i32(keep))
    pool.fork(parent, keep)
    same(p, pool, "fork")
    start, length, want = [-2 ** 31, 0, 5], [96, 2 ** 31 - 1, 5], [96, 2 ** 31 - 1, -2 ** 31]
    assert reserve(p, start, length, want) == pool.reserve(start, length, want)
    same(p, pool, "reserve")
    K.pages_free(p, i32([0, 2 ** 31 - 1, 0]))
    pool.free([0, 2 ** 31 - 1, 0])
    same(p, pool, "free")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n_rows,page,nk", [(1, 16, 1), (7, 64, 4), (64, 16, 2), (65, 32, 1), (256, 256, 3), (257, 16, 2), (900, 64, 1), (400, 16, 12),
                                            (3, 16, 20), (600, 32, 11)])
def test_compact(device, D, n_rows, page, nk):
    """Rows moved over one another, from one slot on to far; sequences that move nothing, or all of theirs by one."""
    print(f"compact D {D} rows {n_rows} page {page} nk {nk}", flush=True)
    rng = np.random.default_rng([D, n_rows, page])
    n, L = 4, 2 * n_rows + 70
    pool = Pool(rng, 3, n * (-(-L // page)) + 2, page, nk, D, n, -(-L // page))
    own_pages(pool, rng, [L] * n)
    first = np.array([3, 0, 50, 20])
    rows = np.stack([f + np.sort(rng.permutation(L - f)[:n_rows]) for f in first])
    rows[2] = first[2] + 1 + np.arange(n_rows)  # all by one
    rows[3] = first[3] + np.arange(n_rows)      # where they are
    counts = np.array([n_rows, max(0, n_rows - 5), n_rows, n_rows])
    for given in (counts, None):
        p = upload(pool)
        K.pages_compact(p, i32(first), i32(rows), n_rows, counts=None if given is None else i32(given))
        after = Pool(np.random.default_rng(0), 3, pool.n_page, page, nk, D, n, pool.n_table)
        after.data, after.table, after.refs = pool.data.copy(), pool.table, pool.refs
        after.compact(first, rows, counts if given is not None else [n_rows] * n)
        same(p, after)


def test_compact_without_pages(device):
    """Rows whose old or new slot has no page stay; counts are held to n_rows."""
    rng = np.random.default_rng(0)
    pool = Pool(rng, 2, 20, 16, 2, 64, 2, 6)
    own_pages(pool, rng, [96, 96])
    pool.table[0, 1], pool.table[0, 4], pool.table[1, 0] = -1, 20, 2 ** 31 - 1
    p = upload(pool)
    first = [10, -20]
    rows = np.stack([10 + np.sort(rng.permutation(200)[:40]), np.arange(40)])
    K.pages_compact(p, i32(first), i32(rows), 40, counts=i32([2 ** 31 - 1, 40]))
    pool.compact(first, rows, [40, 40])
    same(p, pool)
    K.pages_compact(p, i32(first), i32(rows), 40, counts=i32([-1, -2 ** 31]))
    K.pages_compact(p, i32(first), i32(rows), 0)
    same(p, pool)


@pytest.mark.parametrize("D,nk,page,n_layer", [(64, 1, 16, 3), (128, 4, 64, 2), (64, 3, 256, 1), (128, 64, 256, 1)])
def test_copy(device, D, nk, page, n_layer):
    """Pages into another pool and within one; pairs outside either are left out."""
    rng = np.random.default_rng([D, nk, page])
    a, b = (Pool(rng, n_layer, n, page, nk, D, 1, 1) for n in (9, 13))
    p, q = upload(a), upload(b)
    src, dst = [3, 8, 9, -1, 0, 2 ** 31 - 1, 5, 3], [12, 0, 1, 2, 13, 4, -2 ** 31, 7]
    K.pages_copy(q, p, i32(dst), i32(src), len(src))
    for i, j in zip(src, dst):
        if 0 <= i < 9 and 0 <= j < 13:
            b.data[:, j] = a.data[:, i]
    same(q, b)
    same(p, a)
    K.pages_copy(p, p, i32([0, 4]), i32([1, 7]), 2)
    a.data[:, [0, 4]] = a.data[:, [1, 7]]
    K.pages_copy(p, p, i32([0]), i32([1]), 0)
    same(p, a)


def test_offsets_beyond_32_bits(device):
    """Pages 2.4 GB into a layer, layers 2.4 GB apart: rows, attention of one and of many, copied, moved."""
    n_page, page, nk, nh, D, n_layer, T = 60000, 64, 4, 32, 128, 3, 150
    rng = np.random.default_rng(5)
    p = K.KvPages.allocate(n_layer, n_page, page, nk, D, 2, 16)
    refs = np.ones(n_page, np.int32)
    refs[-20:] = 0
    p.refs.upload(refs)
    ws, missing = K.DeviceBuffer(K.pages_workspace(p)), i32([5])
    K.pages_reserve(p, i32([0, 0]), i32([300, 200]), missing, ws)
    table = p.table.download(np.int32).reshape(2, 16)
    assert missing.download(np.int32)[0] == 0
    assert table[0, :5].tolist() == list(range(n_page - 20, n_page - 15)) and table[1, :4].tolist() == list(range(n_page - 15, n_page - 11))
    x = rng.normal(size=(n_layer, 2, 2, 300, nk, D)).astype(np.float32)
    for layer in range(n_layer):
        bufs = [put(a) for a in x[layer]]
        K.pages_store(p, layer, F32, bufs[0], bufs[1], i32([0, 0]), 300, counts=i32([300, 200]))
    held = values(*groups(x.astype(np.float64)))

    def check(s, n, want, what):
        """Slots below n of sequence s hold want [n_layer][2][n][nk][D]."""
        for layer in range(n_layer):
            out = [K.DeviceBuffer(2 * 300 * nk * D * 4) for _ in range(2)]
            K.pages_load(p, layer, F32, out[0], out[1], 300)
            for i in range(2):
                got = out[i].download(np.float32).reshape(2, 300, nk, D)[s, :n]
                assert np.array_equal(got, want[layer, i].astype(np.float32)), (what, layer, i)

    check(0, 300, held[:, :, 0], "rows")
    check(1, 200, held[:, :, 1, :200], "rows")
    kv = [held[2, i].transpose(0, 2, 1, 3) for i in range(2)]
    for rows, prefixes in ((1, [299, 199]), (4, [296, 196]), (T, [150, 50])):
        q = rng.normal(size=(2, rows, nh, D)).astype(np.float32).astype(np.float64)
        got, _ = attend(p, F32, q, rows, prefixes, None, None, nh, layer=2)
        want, bound = tree64(q, kv, prefixes, [rows] * 2, np.stack([np.tril(np.ones((rows, rows), bool))] * 2), D ** -0.5, F32)
        close(got, want, bound, f"{rows} rows")
    # the first sequence's start shared, its third page copied
    K.pages_fork(p, i32([0, 0]), ws, keep=i32([300, 130]))
    K.pages_reserve(p, i32([300, 130]), i32([300, 140]), missing, ws)
    table = p.table.download(np.int32).reshape(2, 16)
    assert table[1, :2].tolist() == table[0, :2].tolist() and table[1, 2] == n_page - 15
    check(1, 130, held[:, :, 0, :130], "copied")
    # 100 of its rows moved together
    moved = np.sort(rng.choice(np.arange(160, 300), 100, False))
    K.pages_compact(p, i32([130, 0]), i32(np.stack([moved, np.arange(100)])), 100, counts=i32([100, 0]))
    now = held[:, :, 0, :230].copy()
    now[:, :, 130:] = held[:, :, 0, moved]
    check(0, 230, now, "moved")
    K.pages_copy(p, p, i32([7, n_page - 1]), i32([n_page - 20, n_page - 19]), 2)
    table[1, :2] = [7, n_page - 1]
    p.table.upload(table)
    check(1, 128, held[:, :, 0, :128], "pages copied")


# ------------------------------------------------------------------ together

class Serving:
    """Sequences of one layer in pages: prompts shared by forking, drafts verified and accepted."""

    def __init__(self, rng, n, nk=2, nh=8, D=64, page=16, T=5, t=F32, stream=None, n_table=20, n_layer=2):
        self.n, self.nk, self.nh, self.D, self.T, self.t, self.stream = n, nk, nh, D, T, t, stream
        self.p = K.KvPages.allocate(n_layer, n * n_table, page, nk, D, n, n_table)
        self.length = np.zeros(n, np.int64)
        self.kv = [np.zeros((n, n_table * page, nk, D)) for _ in range(2)]  # what the cache stands for
        self.missing = i32([0])
        self.ws = K.DeviceBuffer(max(K.pages_workspace(self.p), 1 << 22))
        self.most = n_table * page
        self.keep = []

    def dev(self, a):
        b = i32(a)
        self.keep.append(b)
        return b

    def reserve(self, want, start=None):
        K.pages_reserve(self.p, self.dev(self.length), self.dev(want), self.missing, self.ws, start=start, stream=self.stream)

    def store(self, rng, first, n_rows, counts):
        x = rng.normal(size=(2, self.n, n_rows, self.nk, self.D))
        raw = [encode(a, self.t) for a in x]
        bufs = [put(a) for a in raw]
        self.keep += bufs
        K.pages_store(self.p, 1, self.t, bufs[0], bufs[1], self.dev(first), n_rows, counts=self.dev(counts), stream=self.stream)
        for i in range(2):
            v = values(*groups(decode(raw[i], self.t).reshape(x[i].shape)))
            for s in range(self.n):
                self.kv[i][s, first[s]:first[s] + counts[s]] = v[s, :counts[s]]

    def attend(self, rng, prefix, T, sees):
        q = decode(encode(rng.normal(size=(self.n, T, self.nh, self.D)), self.t), self.t)
        got, _ = attend(self.p, self.t, q, T, prefix, None, sees, self.nh)
        kv = [x.transpose(0, 2, 1, 3) for x in self.kv]
        want, bound = tree64(q, kv, prefix, [T] * self.n, sees, self.D ** -0.5, self.t)
        close(got, want, bound, "serving")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("page", [16, 64])
def test_serving(device, t, page):
    """A prompt shared by four sequences, two steps of drafts verified, accepted and let go, a beam step, a decode step;
    attention after each against float64 over what was stored."""
    rng = np.random.default_rng([t, page])
    z = Serving(rng, 4, page=page, t=t)
    chain = lambda T: np.stack([np.tril(np.ones((T, T), bool))] * 4)  # noqa: E731
    # a prompt of 70 tokens in sequence 2, taken over by all
    want = np.where(np.arange(4) == 2, 70, 0)
    z.reserve(want)
    z.store(rng, np.zeros(4, int), 70, want)
    K.pages_fork(z.p, z.dev([2, 2, 2, 2]), z.ws, keep=z.dev([70, 70, 70, 65]))
    for i in range(2):
        z.kv[i][:] = z.kv[i][2]
    z.length = np.array([70, 70, 70, 65])
    for step in range(2):
        T = z.T
        z.reserve(z.length + T)
        z.store(rng, z.length, T, np.full(4, T))
        sees = np.stack([tree_bits(rng, T) for _ in range(4)])
        z.attend(rng, z.length, T, sees)
        paths = [np.flatnonzero(sees[s, rng.integers(0, T)]) for s in range(4)]  # an accepted row's ancestors and itself
        rows = np.zeros((4, T), int)
        for s in range(4):
            rows[s, :len(paths[s])] = z.length[s] + paths[s]
        counts = np.array([len(a) for a in paths])
        K.pages_compact(z.p, z.dev(z.length), z.dev(rows), T, counts=z.dev(counts))
        K.pages_free(z.p, z.dev(z.length + counts))
        for s in range(4):
            for i in range(2):
                z.kv[i][s, z.length[s]:z.length[s] + counts[s]] = z.kv[i][s, rows[s, :counts[s]]].copy()
        z.length = z.length + counts
    parent = [1, 1, 3, 1]
    K.pages_fork(z.p, z.dev(parent), z.ws, keep=z.dev(z.length[parent]))
    z.length = z.length[parent]
    for i in range(2):
        z.kv[i] = z.kv[i][parent].copy()
    for _ in range(3):
        z.reserve(z.length + 1)
        z.store(rng, z.length, 1, np.ones(4, int))
        z.attend(rng, z.length, 1, chain(1))
        z.length = z.length + 1
    assert z.missing.download(np.int32)[0] == 0
    table, refs = z.p.table.download(np.int32), z.p.refs.download(np.int32)
    assert np.array_equal(np.bincount(table[table >= 0], minlength=refs.size), refs)
    # everything into a larger pool, under the same table
    big = K.KvPages.allocate(2, refs.size + 7, page, z.nk, z.D, 4, z.p.desc.n_table)
    ids = np.arange(refs.size, dtype=np.int32)
    K.pages_copy(big, z.p, z.dev(ids + 7), z.dev(ids), ids.size)
    big.table.upload(np.where(table >= 0, table + 7, -1).astype(np.int32))
    small, z.p = z.p, big
    z.attend(rng, z.length - 1, 1, chain(1))
    # nothing left
    K.pages_free(small, z.dev([0] * 4))
    assert not small.refs.download(np.int32).any() and (small.table.download(np.int32) == -1).all()


class Step:
    """A verify step's calls on given buffers: fork, reserve, store, attention, compact, free."""

    def __init__(self, rng, stream, D, page, T, nh=8, nk=2, n=3):
        self.n, self.T, self.nh, self.D, self.stream = n, T, nh, D, stream
        self.pool = filled(rng, [260] * n, page, nk, D, spare=20 * n)
        self.pool.table[:, -(-260 // page):] = -1
        p = self.p = upload(self.pool)
        self.length = i32([200, 131, 250][:n])
        self.want = i32(np.array([200, 131, 250][:n]) + T)
        self.parent = i32([0, 0, 2][:n])
        self.keep = i32([200, 200, 250][:n])
        self.prefix = i32([200, 200, 250][:n])
        self.wanted = i32(np.array([200, 200, 250][:n]) + T)
        self.x = put(rng.normal(size=(n * T, (nh + 2 * nk) * D)).astype(np.float32))
        self.rows = i32(np.array([200, 200, 250][:n])[:, None] + T - T // 2 + np.arange(T)[None])
        self.counts = i32([T // 2] * n)
        self.left = i32(np.array([200, 200, 250][:n]) + T // 2)
        self.out = K.DeviceBuffer(4 * n * T * nh * D)
        self.missing = i32([5])
        self.ws = K.DeviceBuffer(max(K.pages_workspace(p), 16))
        self.aws = K.DeviceBuffer(max(K.attention_pages_workspace(p, nh, T, 260), 16))
        self.nk = nk
        self.at0 = [self.pool.data, self.pool.table, self.pool.refs]

    def reset(self):
        for b, a in zip((self.p.data, self.p.table, self.p.refs), self.at0):
            b.upload(a)
        self.out.zero()

    def run(self):
        p, s, row = self.p, self.stream, (self.nh + 2 * self.nk) * self.D
        K.pages_fork(p, self.parent, self.ws, keep=self.keep, stream=s)
        K.pages_reserve(p, self.prefix, self.wanted, self.missing, self.ws, stream=s)
        k = self.x.ptr + 4 * self.nh * self.D
        K.pages_store(p, 1, F32, k, k + 4 * self.nk * self.D, self.prefix, self.T, row_stride=row, stream=s)
        K.attention_pages(p, 1, F32, self.x, self.out, self.nh, self.T, self.prefix, 260, self.aws, q_stride=row, stream=s)
        K.pages_compact(p, self.prefix, self.rows, self.T, counts=self.counts, stream=s)
        K.pages_free(p, self.left, stream=s)

    def outputs(self):
        return [self.out.download(np.float32), self.p.data.download(np.uint8), self.p.table.download(np.int32),
                self.p.refs.download(np.int32), self.missing.download(np.int32)]


SHAPES = [dict(D=64, page=16, T=4), dict(D=128, page=64, T=1), dict(D=128, page=128, T=300)]


@pytest.mark.parametrize("pair", [(0, 1), (2, 1)])
def test_two_streams_at_once(streams, pair):
    """Two steps on two streams, workspaces each, give what each gives alone."""
    steps = [Step(np.random.default_rng(i), streams[i], **SHAPES[pair[i]]) for i in range(2)]
    want = []
    for st in steps:
        for _ in range(6):
            st.run()
        K.synchronize()
        want.append(st.outputs())
        st.reset()
    K.synchronize()
    for _ in range(6):
        for st in steps:
            st.run()
    K.synchronize()
    for st, w in zip(steps, want):
        for a, b in zip(st.outputs(), w):
            assert np.array_equal(a, b)


@pytest.mark.parametrize("pair", [(0, 1), (2, 1)])
def test_steps_in_graphs(streams, pair):
    """Captured steps, replayed with inputs changed in between and eager work between replays."""
    h, stream = hip(), streams[0]
    steps = [Step(np.random.default_rng(i), stream, **SHAPES[pair[i]]) for i in range(2)]
    graphs = []
    for st in steps:
        st.run()
        K.synchronize()
        graph, exe = C.c_void_p(), C.c_void_p()
        assert h.hipStreamBeginCapture(stream, 2) == 0  # hipStreamCaptureModeRelaxed
        st.run()
        assert h.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert h.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
        graphs.append((graph, exe))
    rng = np.random.default_rng(9)
    for _ in range(4):
        for st, (_, exe) in zip(steps, graphs):
            prefix = np.full(st.n, rng.integers(40, 250))  # (any sequence may be another's parent)
            for b, a in ((st.prefix, prefix), (st.keep, prefix), (st.wanted, prefix + st.T), (st.left, prefix + st.T // 2),
                         (st.parent, rng.integers(0, st.n, st.n)), (st.rows, prefix[:, None] + st.T - st.T // 2 + np.arange(st.T))):
                b.upload(a.astype(np.int32))
            st.x.upload(rng.normal(size=st.x.nbytes // 4).astype(np.float32))
            st.reset()
            K.synchronize()
            for _ in range(2):
                assert h.hipGraphLaunch(exe, stream) == 0
            K.synchronize()
            got = st.outputs()
            assert np.isfinite(got[0]).all()
            st.reset()
            K.synchronize()
            st.run()
            st.run()
            K.synchronize()
            for a, b in zip(got, st.outputs()):
                assert np.array_equal(a, b)
    for graph, exe in graphs:
        h.hipGraphExecDestroy(exe)
        h.hipGraphDestroy(graph)


def test_wrong_current_device_is_refused(device):
    """The calls run on the opened device only."""
    h, n = hip(), C.c_int()
    assert h.hipGetDeviceCount(C.byref(n)) == 0
    if n.value < 2:
        pytest.skip("one GPU")
    p = K.KvPages.allocate(1, 2, 16, 1, 64, 1, 1)
    assert h.hipSetDevice(1) == 0
    try:
        with pytest.raises(K.KnjError) as e:
            K.pages_free(p, p.refs)
        assert e.value.code == K.KNJ_E_STATE
    finally:
        assert h.hipSetDevice(0) == 0
