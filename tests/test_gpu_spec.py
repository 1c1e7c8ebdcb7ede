"""GPU: the speculative-step operators -- rotary positions, cache rows in f16 and 8
bits, the attention of a tree of drafts, token log probabilities -- against
plain float64 implementations, at the sizes and contents where they can go
wrong, and together as a step uses them."""
import ctypes as C

import numpy as np
import pytest

import kanjoos_amd as K

pytestmark = pytest.mark.gpu

F32, F16, BF16 = K.TYPE_F32, K.TYPE_F16, K.TYPE_BF16
U = 2.0 ** -24                                  # half a step of f32, relative
HALF = {F32: U, F16: 2.0 ** -11, BF16: 2.0 ** -8}  # of an activation's type
TYPES = [F32, F16, BF16]
FORMATS = [K.KV_F16, K.KV_F8, K.KV_I8]


# ------------------------------------------------------------------ host side of the types

def bf16_bits(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def encode(x, t):
    """float64 values as an activation's bytes."""
    x = np.asarray(x)
    with np.errstate(over="ignore"):
        x = x.astype(np.float32)
        return x if t == F32 else x.astype(np.float16) if t == F16 else bf16_bits(x)


def decode(a, t):
    """An activation array as float64."""
    if t == BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def np_type(t):
    return {F32: np.float32, F16: np.float16, BF16: np.uint16}[t]


def put(a):
    return K.DeviceBuffer.from_array(a)


def i32(a):
    return put(np.asarray(a, np.int32))


def close(got, want, bound, what=""):
    """|got - want| <= bound where both are finite; the same infinities and NaN elsewhere."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)]), what
    err, b = np.abs(got[fin] - want[fin]), np.broadcast_to(bound, want.shape)[fin]
    worst = float(np.max(err / np.maximum(b, 1e-300))) if err.size else 0.0
    print(f"{what}: worst error {worst:.3f} of its bound", flush=True)
    assert np.all(err <= b), f"{what}: {worst} of the bound"


# ------------------------------------------------------------------ rotary positions

def rope64(x, w, pos, inv, ms, n_rot, layout, eps):
    """x [rows][heads][D]"""
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    y = x.copy()
    th = np.asarray(pos, np.float64)[:, None] * inv
    c, s = np.cos(th)[:, None] * ms, np.sin(th)[:, None] * ms
    h = n_rot // 2
    a, b = (x[..., :h], x[..., h:n_rot]) if layout == K.ROPE_HALF else (x[..., 0:n_rot:2], x[..., 1:n_rot:2])
    ya, yb = a * c - b * s, a * s + b * c
    if layout == K.ROPE_HALF:
        y[..., :h], y[..., h:n_rot] = ya, yb
    else:
        y[..., 0:n_rot:2], y[..., 1:n_rot:2] = ya, yb
    return y


def rope_bound(want, x, w, ms, t, eps):
    """The norm's sum of 128 squares, its root, quotient and two products (12 U), the
    angle's f32 functions (4 U of 1) and the rotation (4 U), relative to the larger
    of a pair, which a whole head's largest bounds; then the output's own rounding."""
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    big = np.abs(x).max(-1, keepdims=True) * 1.4143 * max(ms, 1.0)
    return 24 * U * big + HALF[t] * np.abs(want) + 1e-30


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("layout", [K.ROPE_HALF, K.ROPE_INTERLEAVED])
@pytest.mark.parametrize("D,n_rot,nh,nk,rows,norm", [
    (128, 128, 32, 4, 1, True), (128, 128, 32, 4, 37, True), (128, 40, 3, 1, 5, False), (128, 8, 17, 0, 2, True),
    (64, 64, 16, 2, 9, False), (64, 24, 5, 5, 3, True), (64, 56, 33, 1, 2, True)])
def test_rope(device, t, layout, D, n_rot, nh, nk, rows, norm):
    print(f"rope type {t} layout {layout} D {D} n_rot {n_rot} heads {nh}/{nk} rows {rows} norm {norm}", flush=True)
    rng = np.random.default_rng([D, n_rot, nh, nk, rows, layout, t])
    stride = (nh + 2 * nk) * D + 24  # rows [q | k | v | pad]
    raw = encode(rng.normal(size=(rows, stride)) * np.exp(rng.normal(size=(rows, 1))), t)
    x = decode(raw, t)
    q, k = x[:, :nh * D].reshape(rows, nh, D), x[:, nh * D:(nh + nk) * D].reshape(rows, nk, D)
    w = [1 + 0.1 * rng.normal(size=D).astype(np.float32) for _ in range(2)]
    pos = rng.integers(0, 40000, rows)
    pos[0], pos[-1] = 0, 1 << 20
    if rows > 2:
        pos[1] = -3
    inv, ms = K.rope_freqs(n_rot, 1e6, K.ROPE_YARN, 4.0, 32768)
    buf, dinv = put(raw), put(inv)
    size = raw.itemsize
    qo, ko = K.DeviceBuffer(rows * nh * D * size), K.DeviceBuffer(max(1, rows * nk * D * size))
    wn = [put(a) if norm else None for a in w]
    args = (t, buf.ptr, buf.ptr + nh * D * size if nk else None, i32(pos), dinv, rows, nh, nk, D)
    kw = dict(n_rot=n_rot, layout=layout, mscale=ms, q_norm=wn[0], k_norm=wn[1], eps=1e-5, q_stride=stride, k_stride=stride)
    K.rope(*args, q_out=qo, k_out=ko if nk else None, **kw)
    for got, x64, wt, n in ((qo, q, w[0], nh), (ko, k, w[1], nk)):
        if n == 0:
            continue
        wt = wt.astype(np.float64) if norm else None
        want = rope64(x64, wt, pos, inv, ms, n_rot, layout, 1e-5)
        g = decode(got.download(np_type(t), rows * n * D), t).reshape(rows, n, D)
        close(g, want, rope_bound(want, x64, wt, ms, t, 1e-5), "q" if n == nh else "k")
    # in place: the same bits, and the rest of the rows untouched
    K.rope(*args, **kw)
    after = buf.download(np_type(t), rows * stride).reshape(rows, stride)
    assert np.array_equal(after[:, :nh * D], qo.download(np_type(t), rows * nh * D).reshape(rows, -1))
    if nk:
        assert np.array_equal(after[:, nh * D:(nh + nk) * D], ko.download(np_type(t), rows * nk * D).reshape(rows, -1))
    assert np.array_equal(after[:, (nh + nk) * D:], raw[:, (nh + nk) * D:])


def test_rope_far_positions(device):
    """Angles of positions near 2^31: cos and sin alone (the pair (1, 0) turned)."""
    D, pos = 64, np.array([2 ** 31 - 1, 2 ** 31 - 2, 123456789, -2 ** 31])
    inv, _ = K.rope_freqs(D, 1e4)
    x = np.zeros((4, 1, D), np.float32)
    x[..., :D // 2] = 1
    out = K.DeviceBuffer(x.nbytes)
    K.rope(F32, put(x), None, i32(pos), put(inv), 4, 1, 0, D, q_out=out)
    th = pos[:, None].astype(np.float64) * inv
    want = np.concatenate([np.cos(th), np.sin(th)], -1)
    # the f64 product and its reduction: 2^31 * 2^-53 each; the f32 functions: 4 U
    close(out.download(np.float32).reshape(4, D), want, 2.0 ** -20 + 4 * U, "far")


# ------------------------------------------------------------------ cache rows

E4M3 = np.array([(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)])
E4M3[127] = np.nan


def codes(x, fmt):
    """Rows x [..., D] (float64 holding f32) as codes (uint8 bit patterns or f16 bits)
    and scales (float32), from the definition: the correctly rounded quotient in
    float64 decides, and is a tie exactly where the quotient is."""
    if fmt == K.KV_F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float32).astype(np.float16).view(np.uint16), None
    top = 127.0 if fmt == K.KV_I8 else 448.0
    amax = np.abs(x).max(-1)
    bad = ~np.isfinite(x).all(-1)
    live = ~bad & (amax >= 2.0 ** -119)
    den = np.where(live, amax, 1.0)[..., None]
    y = np.where(live[..., None], x, 0.0) * top / den
    if fmt == K.KV_I8:
        c = np.rint(y).astype(np.int8).view(np.uint8)
    else:
        step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
        v = np.rint(y / step) * step
        c = np.searchsorted(E4M3[:127], np.abs(v)).astype(np.uint8)
        assert np.array_equal(E4M3[c], np.abs(v))
        c |= (np.signbit(y) * 128).astype(np.uint8)
    s = np.where(bad, np.nan, np.where(live, amax.astype(np.float32) / np.float32(top), 0)).astype(np.float32)
    return c, s


def values(c, s, fmt):
    """Codes and scales as float64."""
    if fmt == K.KV_F16:
        return c.view(np.float16).astype(np.float64)
    v = c.view(np.int8).astype(np.float64) if fmt == K.KV_I8 else E4M3[c & 127] * np.where(c & 128, -1.0, 1.0)
    with np.errstate(invalid="ignore"):
        return v * s[..., None].astype(np.float64)


def cache_arrays(c):
    """A cache's buffers as arrays [n_seq][n_head_kv][n_ctx](D); padding between sequences dropped."""
    d = c.desc
    per = d.seq_stride or d.n_head_kv * d.n_ctx * d.head_dim
    n = d.n_head_kv * d.n_ctx
    dt = np.uint16 if d.format == K.KV_F16 else np.uint8
    out = {}
    for m in ("k", "v"):
        a = getattr(c, m).download(dt, d.n_seq * per).reshape(d.n_seq, per)[:, :n * d.head_dim]
        out[m] = a.reshape(d.n_seq, d.n_head_kv, d.n_ctx, d.head_dim)
        if d.format != K.KV_F16:
            s = getattr(c, m + "_scale").download(np.float32, d.n_seq * per // d.head_dim)
            out[m + "_scale"] = s.reshape(d.n_seq, -1)[:, :n].reshape(d.n_seq, d.n_head_kv, d.n_ctx)
        else:
            out[m + "_scale"] = None
    return out


def make_cache(fmt, n_seq, nk, n_ctx, D, pad=0, fill=0):
    """A cache with `pad` slots' room between sequences, its bytes `fill`."""
    per = (nk * n_ctx + pad) * D
    eb = 2 if fmt == K.KV_F16 else 1
    bufs = [put(np.full(n_seq * per * eb, fill, np.uint8)) for _ in range(2)]
    bufs += [None, None] if fmt == K.KV_F16 else [put(np.full(n_seq * per // D * 4, fill, np.uint8)) for _ in range(2)]
    return K.KvCache(fmt, n_seq, nk, n_ctx, D, *bufs, seq_stride=per if pad else 0)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,nk,n_seq,rows,pad", [(128, 4, 1, 1, 0), (128, 1, 3, 11, 5), (64, 3, 2, 65, 0), (64, 8, 5, 2, 3)])
def test_kv_store_load(device, t, fmt, D, nk, n_seq, rows, pad):
    """Codes and scales bit for bit, values read back to their rounding; rows past the
    counts and slots outside the cache neither written nor read."""
    print(f"kv type {t} format {fmt} D {D} heads {nk} seqs {n_seq} rows {rows}", flush=True)
    rng = np.random.default_rng([D, nk, n_seq, rows, fmt, t])
    n_ctx, stride = rows + 7, 2 * nk * D + 8
    raw = encode(rng.normal(size=(n_seq * rows, stride)) * np.exp(2 * rng.normal(size=(n_seq * rows, 1))), t)
    if rows > 10:  # a row of zeros, a tiny one, halves of the largest (ties), an infinity, a NaN
        raw[0] = 0
        raw[1] = encode(rng.normal(size=stride) * 1e-38, t)
        raw[2] = encode(rng.choice([1.0, -0.5, 0.5, 0.25, 1.5 / 127, 0.5 / 448 * 2 ** -9], stride), t)
        raw[3, 5] = encode([np.inf], t)[0]
        raw[4, 9] = encode([np.nan], t)[0]
        raw[4, nk * D + 1] = encode([np.nan], t)[0]
    x = decode(raw, t).reshape(n_seq, rows, stride)
    start = rng.integers(0, 8, n_seq)
    counts = rng.integers(0, rows + 1, n_seq)
    counts[0] = rows + 9  # held to the rows there are
    if n_seq > 2:
        start[1], start[2] = -1, n_ctx - 1
        counts[1:3] = rows
    if n_seq > 4:
        start[4], counts[3], counts[4] = 2 ** 31 - 1, -5, rows
    c = make_cache(fmt, n_seq, nk, n_ctx, D, pad, fill=0x11)
    before = cache_arrays(c)
    buf = put(raw)
    K.kv_store(c, t, buf.ptr, buf.ptr + nk * D * raw.itemsize, i32(start), rows, counts=i32(counts), row_stride=stride)
    after = cache_arrays(c)
    want = {m: (None if a is None else a.copy()) for m, a in before.items()}
    for m, off in (("k", 0), ("v", nk * D)):
        code, scale = codes(x[..., off:off + nk * D].reshape(n_seq, rows, nk, D), fmt)
        for s in range(n_seq):
            for i in range(rows):
                slot = int(start[s]) + i
                if i < counts[s] and 0 <= slot < n_ctx:
                    want[m][s, :, slot] = code[s, i]
                    if scale is not None:
                        want[m + "_scale"][s, :, slot] = scale[s, i]
        if fmt == K.KV_F16:
            nan = np.isnan(want[m].view(np.float16))
            assert np.array_equal(nan, np.isnan(after[m].view(np.float16)))
            assert np.array_equal(after[m][~nan], want[m][~nan])
        else:
            assert np.array_equal(after[m], want[m])
            np.testing.assert_array_equal(after[m + "_scale"], want[m + "_scale"])
    # read back, some rows from outside the cache
    slots = rng.integers(0, n_ctx, (n_seq, rows))
    slots[0, 0] = -1 if rows > 1 else 0
    slots[-1, -1] = n_ctx
    mark = encode(np.full((n_seq * rows, nk * D + 8), 7.0), t)
    out = [put(mark), put(mark)]
    K.kv_load(c, t, out[0], out[1], rows, slots=i32(slots), row_stride=nk * D + 8)
    for m, o in zip(("k", "v"), out):
        got = o.download(np_type(t), mark.size).reshape(n_seq, rows, -1)
        v = values(after[m], after[m + "_scale"], fmt)
        for s in range(n_seq):
            inside = (slots[s] >= 0) & (slots[s] < n_ctx)
            w = v[s][:, slots[s][inside]].transpose(1, 0, 2).reshape(-1, nk * D)
            with np.errstate(over="ignore", invalid="ignore"):
                w = np.where(np.abs(w) > 65519 * 1.0001, np.sign(w) * np.inf, w) if t == F16 else w
            close(decode(got[s][inside][:, :nk * D], t), w, (U + HALF[t]) * np.abs(w) + (2.0 ** -25 if t == F16 else 2e-45 + 1e-40 * (t == BF16)), m)
            keep = np.ones(got[s].shape, bool)
            keep[inside, :nk * D] = False
            assert np.array_equal(got[s][keep], np.broadcast_to(mark[0], got[s].shape)[keep])
    # the whole cache by slot number
    if n_ctx >= rows:
        K.kv_load(c, F32, *(big := [K.DeviceBuffer(4 * n_seq * rows * nk * D) for _ in range(2)]), rows)
        got = big[0].download(np.float32).reshape(n_seq, rows, nk, D).astype(np.float64)
        v = values(after["k"], after["k_scale"], fmt)[:, :, :rows].transpose(0, 2, 1, 3)
        close(got, v, U * np.abs(v) + 1e-45, "by slot")


@pytest.mark.parametrize("fmt", FORMATS)
def test_kv_move_keeps_codes(device, fmt):
    """Rows loaded as f32 and stored again keep their codes; their scales move by a rounding or two."""
    rng = np.random.default_rng(fmt)
    D, nk, rows = 128, 4, 64
    c, c2 = K.KvCache.allocate(fmt, 1, nk, rows, D), K.KvCache.allocate(fmt, 1, nk, rows, D)
    x = put((rng.normal(size=(rows, 2, nk * D)) * np.exp(3 * rng.normal(size=(rows, 2, 1)))).astype(np.float32))
    zero = i32([0])
    K.kv_store(c, F32, x.ptr, x.ptr + 4 * nk * D, zero, rows, row_stride=2 * nk * D)
    f = [K.DeviceBuffer(4 * rows * nk * D) for _ in range(2)]
    K.kv_load(c, F32, f[0], f[1], rows)
    K.kv_store(c2, F32, f[0], f[1], zero, rows)
    a, b = cache_arrays(c), cache_arrays(c2)
    for m in ("k", "v"):
        assert np.array_equal(a[m], b[m])
        if fmt != K.KV_F16:
            np.testing.assert_allclose(a[m + "_scale"], b[m + "_scale"], rtol=3 * 2 * U)


# ------------------------------------------------------------------ the drafts' attention

def tree_bits(rng, T, chain=False):
    """[T][T] truth values: ancestors and itself."""
    sees = np.zeros((T, T), bool)
    for t in range(T):
        if t:
            p = t - 1 if chain or rng.random() < 0.5 else int(rng.integers(0, t))
            sees[t] = sees[p]
        sees[t, t] = True
    return sees


def mask_words(sees):
    """[...][T][T] truth values as 64-bit words [...][T][ceil(T/64)]."""
    T = sees.shape[-1]
    bits = np.zeros(sees.shape[:-1] + ((T + 63) // 64 * 64,), bool)
    bits[..., :T] = sees
    return np.packbits(bits, axis=-1, bitorder="little").view(np.uint64)


def tree64(q, kv, prefix, counts, sees, scale, t):
    """Attention in float64 and its error bound.  q [n][T][nh][D]; kv two arrays
    [n][nk][ctx][D].  With A the largest scale |q|.|k| of the slots a row sees: a
    score is off by 16 U A (128 products summed pairwise within the matrix core,
    the queries' 22 bits, the exponent's argument), a weight by that twice over
    and 64 U, with 16-bit activations by their 11 bits; a weight far below the
    largest is held to 2^-25 of it, at random: six standard deviations of the sum."""
    n, T, nh, D = q.shape
    nk = kv[0].shape[1]
    out, bound = np.full(q.shape, np.nan), np.zeros(q.shape)
    w_half = 0.0 if t == F32 else 2.0 ** -11
    for s in range(n):
        P, N = int(prefix[s]), int(counts[s])
        for h in range(nh):
            kk, vv = kv[0][s, h * nk // nh], kv[1][s, h * nk // nh]
            for i in range(N):
                slots = np.concatenate([np.arange(P), P + np.nonzero(sees[s, i, :N])[0]]).astype(int)
                if slots.size == 0:
                    out[s, i, h] = 0
                    continue
                ks, vs = kk[slots], vv[slots]
                if not np.isfinite(vs[slots >= P]).all():
                    continue  # NaN
                sc = scale * (ks @ q[s, i, h])
                A = scale * (np.abs(ks) @ np.abs(q[s, i, h])).max()
                p = np.exp(sc - sc.max())
                l = p.sum()
                p /= l
                out[s, i, h] = p @ vs
                rms = np.sqrt((vs ** 2).sum(0))
                bound[s, i, h] = (32 * U * A + 64 * U + w_half) * (p @ np.abs(vs)) + 6 * 2.0 ** -25 * rms / l \
                    + HALF[t] * np.abs(out[s, i, h]) + (2.0 ** -25 if t == F16 else 1e-37)
    return out, bound


def run_tree(c, t, q, T, prefix, counts, sees, nh, max_prefix=None, shared=False, scale=None, pad=0, in_place=False):
    """attention_tree on host arrays; rows of q and out `pad` elements apart."""
    n, D = c.desc.n_seq, c.desc.head_dim
    width = nh * D
    rows = np.full((n * T, width + pad), 7.0)
    mark = encode(rows, t)
    rows[:, :width] = q.reshape(n * T, width)
    dq = put(encode(rows, t))
    out = dq if in_place else put(mark)
    max_prefix = int(max(prefix)) if max_prefix is None else max_prefix
    ws = K.DeviceBuffer(K.attention_tree_workspace(c, nh, T, max_prefix) + 64)
    ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))  # NaN wherever nothing is written
    K.attention_tree(c, t, dq, out, nh, T, i32(prefix), max_prefix, ws, counts=None if counts is None else i32(counts),
                     mask=None if sees is None else put(mask_words(sees)), mask_shared=shared, scale=scale,
                     q_stride=width + pad, out_stride=width + pad)
    got = out.download(np_type(t), mark.size).reshape(n * T, -1)
    base = encode(rows, t) if in_place else mark
    assert np.array_equal(got[:, width:], base[:, width:])
    return decode(got[:, :width], t).reshape(n, T, nh, D), decode(base[:, :width], t).reshape(n, T, nh, D)


def fill_cache(c, rng, spread=0.5):
    """Random rows in every slot of every sequence; returns their values [n][nk][ctx][D]."""
    d = c.desc
    shape = (d.n_seq, d.n_ctx, d.n_head_kv, d.head_dim)
    kv = [rng.normal(size=shape) * np.exp(spread * rng.normal(size=shape[:3]))[..., None] for _ in range(2)]
    bufs = [put(a.astype(np.float32)) for a in kv]
    K.kv_store(c, F32, bufs[0], bufs[1], i32(np.zeros(d.n_seq)), d.n_ctx)
    a = cache_arrays(c)
    return [values(a[m], a[m + "_scale"], d.format) for m in ("k", "v")]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,nh,nk,T,prefixes", [
    (128, 32, 4, 1, (0, 1, 31, 32, 63)), (128, 8, 1, 2, (64, 65, 126, 127, 128, 129)), (128, 12, 4, 5, (0, 3, 200, 383)),
    (128, 4, 4, 16, (1, 500)), (64, 14, 2, 9, (0, 64, 130)), (64, 16, 2, 3, (1000, 7)), (128, 10, 2, 13, (250, 64)),
    (64, 8, 8, 66, (70, 0)), (128, 24, 1, 7, (129, 300)), (128, 32, 4, 25, (190,))])
def test_attention_tree(device, t, fmt, D, nh, nk, T, prefixes):
    """Trees over prefixes on both sides of the tiles' borders, every column-tile
    shape, groups that are no power of two, sequences of different lengths."""
    print(f"tree type {t} format {fmt} D {D} heads {nh}/{nk} T {T} prefixes {prefixes}", flush=True)
    rng = np.random.default_rng([D, nh, nk, T, fmt, t])
    n = len(prefixes)
    c = make_cache(fmt, n, nk, max(prefixes) + T + 3, D, pad=2)
    kv = fill_cache(c, rng)
    sees = np.stack([tree_bits(rng, T) for _ in range(n)])
    counts = np.array([max(1, T - s % 3) for s in range(n)])
    q = decode(encode(1.5 * rng.normal(size=(n, T, nh, D)), t), t)
    got, before = run_tree(c, t, q, T, prefixes, counts, sees, nh, pad=16)
    want, bound = tree64(q, kv, prefixes, counts, sees, D ** -0.5, t)
    for s in range(n):
        close(got[s, :counts[s]], want[s, :counts[s]], bound[s, :counts[s]], f"prefix {prefixes[s]}")
        assert np.array_equal(got[s, counts[s]:], before[s, counts[s]:])  # rows past the drafts
    # in place
    again, _ = run_tree(c, t, q, T, prefixes, counts, sees, nh, pad=16, in_place=True)
    for s in range(n):
        assert np.array_equal(again[s, :counts[s]], got[s, :counts[s]])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T", [1, 40, 64, 65, 130])
def test_attention_tree_chain(device, fmt, T):
    """No mask: draft t sees drafts 0..t.  The same bits as with the chain's mask, its
    own per sequence or one shared."""
    print(f"chain format {fmt} T {T}", flush=True)
    rng = np.random.default_rng([fmt, T])
    nh, nk, D, prefixes = 6, 2, 128, [0, 77]
    c = make_cache(fmt, 2, nk, 77 + T, D)
    kv = fill_cache(c, rng)
    q = rng.normal(size=(2, T, nh, D)).astype(np.float32).astype(np.float64)
    sees = np.stack([np.tril(np.ones((T, T), bool))] * 2)
    got, _ = run_tree(c, F32, q, T, prefixes, None, None, nh)
    want, bound = tree64(q, kv, prefixes, [T, T], sees, D ** -0.5, F32)
    close(got, want, bound, "chain")
    assert np.array_equal(run_tree(c, F32, q, T, prefixes, None, sees, nh)[0], got)
    assert np.array_equal(run_tree(c, F32, q, T, prefixes, None, sees[:1], nh, shared=True)[0], got)
    # a bound on the prefixes above them changes the split, not the result beyond rounding
    c2 = make_cache(fmt, 2, nk, 5000, D)
    rng = np.random.default_rng([fmt, T])
    kv2 = fill_cache(c2, rng)
    got, _ = run_tree(c2, F32, q, T, prefixes, None, None, nh, max_prefix=4000)
    want, bound = tree64(q, kv2, prefixes, [T, T], sees, D ** -0.5, F32)
    close(got, want, bound, "loose bound")


@pytest.mark.parametrize("fmt", FORMATS)
def test_attention_tree_lengths_held(device, fmt):
    """Prefixes and counts outside their range are held to it."""
    rng = np.random.default_rng(fmt)
    nh, nk, D, T = 4, 2, 64, 3
    c = make_cache(fmt, 5, nk, 100, D)
    kv = fill_cache(c, rng)
    q = rng.normal(size=(5, T, nh, D)).astype(np.float32).astype(np.float64)
    sees = np.stack([tree_bits(rng, T) for _ in range(5)])
    got, before = run_tree(c, F32, q, T, [-7, 5000, 2 ** 31 - 1, 20, -2 ** 31], [T, 2 ** 31 - 1, T, -1, 0], sees, nh, max_prefix=90)
    held, counts = [0, 90, 90, 20, 0], [T, T, T, 0, 0]
    want, bound = tree64(q, kv, held, counts, sees, D ** -0.5, F32)
    for s in range(5):
        close(got[s, :counts[s]], want[s, :counts[s]], bound[s, :counts[s]], f"sequence {s}")
        assert np.array_equal(got[s, counts[s]:], before[s, counts[s]:])


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,nh", [(6, 2), (6, 8), (20, 4), (40, 8)])
def test_attention_tree_unseen_slots(device, t, fmt, T, nh):
    """Slots that a draft does not see count for nothing, whatever they hold: NaN,
    infinities and huge values in unseen drafts' rows and past the drafts; a row
    that sees nothing gives zeros; one that sees a spoilt value gives NaN."""
    print(f"unseen type {t} format {fmt} T {T} heads {nh}", flush=True)
    rng = np.random.default_rng([t, fmt, T])
    nk, D, prefixes = 2, 64, np.array([0, 61, 128])
    c = make_cache(fmt, 3, nk, 200, D)
    fill_cache(c, rng)
    # the drafts: one huge, one with an infinity, one with a NaN, one tiny
    x = rng.normal(size=(2, 3, T, nk, D))
    x[:, :, 1] *= 1e4
    x[1, :, 2, :, 5] = np.inf
    x[0, :, 2, :, 7] = -np.inf
    x[:, :, 3, :, 0] = np.nan
    x[:, :, 4] *= 1e-3
    bufs = [put(a.astype(np.float32)) for a in x]
    K.kv_store(c, F32, bufs[0], bufs[1], i32(prefixes), T)
    # slots past the drafts: every byte of codes and scales set (NaN in each format but int8)
    for s in range(3):
        for m in ("k", "v"):
            for name, eb in ((m, D * (2 if fmt == K.KV_F16 else 1)), (m + "_scale", 4)):
                b = getattr(c, name)
                if b is None:
                    continue
                for h in range(nk):
                    first = (s * nk + h) * 200 + prefixes[s] + T
                    K.check(K.lib().knj_memcpy_h2d(b.ptr + int(first) * eb, K._ptr(np.full((200 - prefixes[s] - T) * eb, 0xFF, np.uint8)),
                                                   int(200 - prefixes[s] - T) * eb))
    a = cache_arrays(c)
    with np.errstate(invalid="ignore"):
        kv = [values(a[m], a[m + "_scale"], fmt) for m in ("k", "v")]
    sees = np.zeros((3, T, T), bool)
    for i in range(T):
        sees[:, i, i] = i not in (1, 2, 3)
        sees[:, i, 0] = True
    sees[:, 0] = False           # nothing but the prefix: nothing at all with a prefix of 0
    sees[:, 5, 4] = True
    sees[0, 2, 2] = sees[1, 2, 3] = True  # a spoilt value seen
    q = decode(encode(rng.normal(size=(3, T, nh, D)), t), t)
    got, _ = run_tree(c, t, q, T, prefixes, None, sees, nh)
    with np.errstate(invalid="ignore", over="ignore"):
        want, bound = tree64(q, kv, prefixes, [T] * 3, sees, D ** -0.5, t)
    assert np.all(want[0, 0] == 0) and np.isnan(want[0, 2]).all() and np.isnan(want[1, 2]).all()
    close(got, want, bound, "unseen")
    assert np.all(got[0, 0] == 0)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("size", [1e-12, 1e-4, 1.0, 3e4, 1e9])
def test_attention_tree_magnitudes(device, fmt, size):
    """Queries of any size against keys whose scores stay ordinary, and 8-bit values of
    any unit: the power-of-two factors are exact."""
    rng = np.random.default_rng(fmt)
    nh, nk, D, T = 8, 2, 128, 4
    c = make_cache(fmt, 1, nk, 300, D)
    shape = (300, nk, D)
    ksize, vsize = (1.0, 1.0) if fmt == K.KV_F16 else (1.0 / size, size)
    bufs = [put((rng.normal(size=shape) * z * np.exp(rng.normal(size=shape[:2]))[..., None]).astype(np.float32)) for z in (ksize, vsize)]
    K.kv_store(c, F32, bufs[0], bufs[1], i32([0]), 300)
    a = cache_arrays(c)
    kv = [values(a[m], a[m + "_scale"], fmt) for m in ("k", "v")]
    q = (rng.normal(size=(1, T, nh, D)) * (1.0 if fmt == K.KV_F16 else size)).astype(np.float32).astype(np.float64)
    scale = D ** -0.5
    if fmt == K.KV_F16:  # the scale takes the size out again where it may
        q, scale = (q * size).astype(np.float32).astype(np.float64), min(1e6, max(1e-6, scale / size))
    sees = np.stack([tree_bits(rng, T)])
    got, _ = run_tree(c, F32, q, T, [290], None, sees, nh, scale=scale)
    scale = float(np.float32(scale))
    want, bound = tree64(q, kv, [290], [T], sees, scale, F32)
    close(got, want, bound, f"size {size}")


def store_prefix(c, kv, n):
    """Rows [n_seq][n][nk][D] (float64) into the first n slots; their values as the cache holds them,
    [n_seq][nk][n][D]."""
    d = c.desc
    bufs = [put(a.astype(np.float32)) for a in kv]
    K.kv_store(c, F32, bufs[0], bufs[1], i32(np.zeros(d.n_seq)), n)
    out = []
    for a in kv:
        code, scale = codes(a.astype(np.float32).astype(np.float64), d.format)
        out.append(values(code, scale, d.format).transpose(0, 2, 1, 3))
    return out


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D,T,nh", [(128, 8, 48), (128, 20, 64), (64, 9, 40), (64, 33, 64)])
def test_attention_tree_wide(device, t, fmt, D, T, nh):
    """The column tiles of 64 and 128 that much work is given to: the bound on the
    prefixes makes the work large, the prefixes themselves stay short."""
    print(f"wide type {t} format {fmt} D {D} T {T} heads {nh}", flush=True)
    rng = np.random.default_rng([t, fmt, D, T])
    n, nk, bound_p = 8, 8, 6000
    c = K.KvCache.allocate(fmt, n, nk, bound_p + T, D)
    prefixes = np.array([0, 63, 64, 129, 300, 1000, 17, 700])
    filled = 1000 + T
    kv = store_prefix(c, [rng.normal(size=(n, filled, nk, D)) * np.exp(0.3 * rng.normal(size=(n, filled, nk)))[..., None] for _ in range(2)],
                      filled)
    sees = np.stack([tree_bits(rng, T) for _ in range(n)])
    counts = np.array([T, T - 1, 1, T, 2, T, 0, T])
    q = decode(encode(1.5 * rng.normal(size=(n, T, nh, D)), t), t)
    got, before = run_tree(c, t, q, T, prefixes, counts, sees, nh, max_prefix=bound_p)
    want, bound = tree64(q, kv, prefixes, counts, sees, D ** -0.5, t)
    for s in range(n):
        close(got[s, :counts[s]], want[s, :counts[s]], bound[s, :counts[s]], f"prefix {prefixes[s]}")
        assert np.array_equal(got[s, counts[s]:], before[s, counts[s]:])


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,nh", [(1, 4), (3, 16), (12, 16)])
@pytest.mark.parametrize("rising", [1, -1])
def test_attention_tree_drifting(device, t, fmt, T, nh, rising):
    """Scores and value units that rise (or fall) along the prefix, so that every
    chunk passes (or none reaches) what the chunks before it left as reference."""
    print(f"drift type {t} format {fmt} T {T} heads {nh} rising {rising}", flush=True)
    rng = np.random.default_rng([t, fmt, T])
    nk, D, P = 2, 128, 1500
    c = make_cache(fmt, 1, nk, P + T, D)
    ramp = np.linspace(0, 1, P + T)[::rising]
    base = rng.normal(size=(nk, D))
    k = (0.2 * rng.normal(size=(1, P + T, nk, D)) + 3 * ramp[None, :, None, None] * base[None, None])
    v = rng.normal(size=(1, P + T, nk, D)) * np.exp2(12 * ramp)[None, :, None, None]
    kv = store_prefix(c, [k, v], P + T)
    sees = tree_bits(rng, T)[None]
    q = 2.0 * np.repeat(base, nh // nk, axis=0)[None, None] + 0.3 * rng.normal(size=(1, T, nh, D))
    q = decode(encode(q, t), t)
    got, _ = run_tree(c, t, q, T, [P], None, sees, nh)
    want, bound = tree64(q, kv, [P], [T], sees, D ** -0.5, t)
    close(got, want, bound, "drift")


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("part", ["k", "v"])
def test_attention_tree_nan_in_prefix(device, fmt, part):
    """A NaN that every draft sees reaches every draft -- of a value in f16 its own
    dim -- and the call ends."""
    rng = np.random.default_rng(fmt)
    nh, nk, D, T, P = 8, 2, 64, 5, 700
    c = make_cache(fmt, 2, nk, P + T, D)
    x = [rng.normal(size=(2, P + T, nk, D)) for _ in range(2)]
    x[part == "v"][1, 400, :, 9] = np.nan
    with np.errstate(invalid="ignore"):
        kv = store_prefix(c, x, P + T)
        q = rng.normal(size=(2, T, nh, D)).astype(np.float32).astype(np.float64)
        sees = np.stack([tree_bits(rng, T)] * 2)
        got, _ = run_tree(c, F32, q, T, [P, P], None, sees, nh)
        want, bound = tree64(q, kv, [P, P], [T, T], sees, D ** -0.5, F32)
    assert np.isnan(want[1, ..., 9]).all() and np.isfinite(want[0]).all()
    close(got, want, np.where(np.isnan(bound), 1.0, bound), "nan")


@pytest.mark.parametrize("fmt", FORMATS)
def test_attention_tree_zero_rows(device, fmt):
    """A prefix of zero rows (scales of zero in 8 bits) that ends in ordinary ones: the
    zeros take their equal part of the weights."""
    rng = np.random.default_rng([19, fmt])
    nh, nk, D, T, P = 8, 2, 64, 2, 400
    c = make_cache(fmt, 1, nk, P + T, D)
    x = rng.normal(size=(2, P + T, nk, D)).astype(np.float32)
    x[:, :300] = 0
    bufs = [put(a) for a in x]
    K.kv_store(c, F32, bufs[0], bufs[1], i32([0]), P + T)
    a = cache_arrays(c)
    kv = [values(a[m], a[m + "_scale"], fmt) for m in ("k", "v")]
    q = rng.normal(size=(1, T, nh, D)).astype(np.float32).astype(np.float64)
    sees = tree_bits(rng, T)[None]
    for prefix in (P, 200):  # the second sees zeros alone before its drafts' slots, which hold zeros too
        got, _ = run_tree(c, F32, q, T, [prefix], None, sees, nh, max_prefix=P)
        want, bound = tree64(q, kv, [prefix], [T], sees, D ** -0.5, F32)
        close(got, want, bound, f"prefix {prefix}")


def test_attention_tree_long_cache(device):
    """Sequences whose cache begins past 2^32 elements."""
    rng = np.random.default_rng(1)
    nh, nk, D, T, n_ctx = 4, 2, 128, 3, 150
    stride = (1 << 32) // D * D + 5 * D
    bufs = [K.DeviceBuffer(stride + nk * n_ctx * D) for _ in range(2)]
    bufs += [K.DeviceBuffer(4 * (stride // D + nk * n_ctx)) for _ in range(2)]
    c = K.KvCache(K.KV_I8, 2, nk, n_ctx, D, *bufs, seq_stride=stride)
    x = [rng.normal(size=(2, n_ctx, nk, D)).astype(np.float32) for _ in range(2)]
    d = [put(a) for a in x]
    K.kv_store(c, F32, d[0], d[1], i32([0, 0]), n_ctx)
    back = [K.DeviceBuffer(x[0].nbytes) for _ in range(2)]
    K.kv_load(c, F32, back[0], back[1], n_ctx)
    kv = []
    for a, b in zip(x, back):
        code, scale = codes(a.astype(np.float64), K.KV_I8)
        v = values(code, scale, K.KV_I8)
        close(b.download(np.float32).reshape(v.shape), v, U * np.abs(v), "rows")
        kv.append(v.transpose(0, 2, 1, 3))
    q = rng.normal(size=(2, T, nh, D)).astype(np.float32).astype(np.float64)
    sees = np.stack([tree_bits(rng, T)] * 2)
    got, _ = run_tree(c, F32, q, T, [140, 147], None, sees, nh)
    want, bound = tree64(q, kv, [140, 147], [T, T], sees, D ** -0.5, F32)
    close(got, want, bound, "far sequence")


def test_attention_tree_first_rows_of_many(device):
    """The largest draft count, with every column-tile shape's remainder."""
    rng = np.random.default_rng(5)
    nh, nk, D, T = 2, 1, 64, 1024
    c = make_cache(K.KV_F8, 1, nk, 1100, D)
    kv = fill_cache(c, rng)
    q = rng.normal(size=(1, T, nh, D)).astype(np.float32).astype(np.float64)
    sees = tree_bits(rng, T)[None]
    for count in (1024, 1000, 33):
        got, before = run_tree(c, F32, q, T, [70], [count], sees, nh)
        want, bound = tree64(q, kv, [70], [count], sees, D ** -0.5, F32)
        close(got[0, :count], want[0, :count], bound[0, :count], f"{count} drafts")
        assert np.array_equal(got[0, count:], before[0, count:])


def test_attention_tree_many_units(device):
    """More (sequence, kv head) pairs than one dimension of the grid holds in eights:
    every pair of 4100 sequences of 64 heads gets its own answer."""
    rng = np.random.default_rng(11)
    n, nk, D, ctx = 4100, 64, 64, 3
    c = make_cache(K.KV_F16, n, nk, ctx, D)
    kv = fill_cache(c, rng)
    prefix = rng.integers(0, ctx, n)
    q = rng.normal(size=(n, 1, nk, D)).astype(np.float16).astype(np.float64)
    got, _ = run_tree(c, F16, q, 1, prefix, None, None, nk, max_prefix=ctx - 1)
    sc = np.einsum("shd,shjd->shj", q[:, 0], kv[0]) * D ** -0.5  # (a chain of one: slots up to its own)
    A = np.einsum("shd,shjd->shj", np.abs(q[:, 0]), np.abs(kv[0])).max(-1) * D ** -0.5
    seen = np.arange(ctx) <= prefix[:, None]
    sc = np.where(seen[:, None], sc, -np.inf)
    e = np.exp(sc - sc.max(-1, keepdims=True))
    l = e.sum(-1, keepdims=True)
    w = e / l
    want = np.einsum("shj,shjd->shd", w, kv[1])
    rms = np.sqrt(np.einsum("shj,shjd->shd", np.broadcast_to(seen[:, None], w.shape).astype(np.float64), kv[1] ** 2))
    # (tree64's bound)
    bound = (32 * U * A[..., None] + 64 * U + 2.0 ** -11) * np.einsum("shj,shjd->shd", w, np.abs(kv[1])) \
        + 6 * 2.0 ** -25 * rms / l + HALF[F16] * np.abs(want) + 2.0 ** -25
    close(got[:, 0], want, bound, "pairs")


@pytest.mark.parametrize("fmt", FORMATS)
def test_attention_tree_many_heads(device, fmt):
    """The most query heads over one kv head."""
    rng = np.random.default_rng([13, fmt])
    nh, D, T, P = 1024, 64, 3, 70
    c = make_cache(fmt, 1, 1, P + T, D)
    kv = fill_cache(c, rng)
    q = rng.normal(size=(1, T, nh, D)).astype(np.float32).astype(np.float64)
    sees = tree_bits(rng, T)[None]
    got, _ = run_tree(c, F32, q, T, [P], None, sees, nh)
    want, bound = tree64(q, kv, [P], [T], sees, D ** -0.5, F32)
    close(got, want, bound, "heads")


@pytest.mark.parametrize("fmt", FORMATS)
def test_kv_rows_of_most_sequences(device, fmt):
    """The most sequences a cache may have, a row each; read back by a slot list that
    names the same slot twice."""
    rng = np.random.default_rng([17, fmt])
    n, D = 65535, 64
    c = make_cache(fmt, n, 1, 1, D)
    x = rng.normal(size=(2, n, D)).astype(np.float32)
    buf = [put(a) for a in x]
    K.kv_store(c, F32, buf[0], buf[1], i32(np.zeros(n)), 1)
    out = [K.DeviceBuffer(2 * x[0].nbytes) for _ in range(2)]
    K.kv_load(c, F32, out[0], out[1], 2, slots=i32(np.zeros(2 * n)))
    for a, o in zip(x, out):
        code, scale = codes(a.astype(np.float64), fmt)
        v = values(code, scale, fmt)[:, None]
        close(o.download(np.float32).reshape(n, 2, D), np.broadcast_to(v, (n, 2, D)), U * np.abs(v) + 1e-45, "rows")


# ------------------------------------------------------------------ log probabilities

def logprobs64(x, tokens, n_top, T):
    """x [rows][vocab] float64 -> logprob, entropy, top indices and log probabilities.
    NaN ranks as -inf."""
    rows, V = x.shape
    raw = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-raw, axis=-1, kind="stable")[:, :n_top]
    lp, ent, top = np.empty(rows), np.empty(rows), np.empty((rows, n_top))
    for r in range(rows):
        if np.isnan(x[r]).any() or (x[r] == np.inf).any():
            logp, ent[r] = np.full(V, np.nan), np.nan
        elif (x[r] == -np.inf).all():
            logp, ent[r] = np.full(V, -np.inf), 0.0
        else:
            d = (x[r] - x[r].max()) / T
            e = np.exp(d)
            first = int(np.argmax(x[r]))
            rest = np.delete(e, first).sum()  # log(1 + rest) keeps a small rest
            logp = d - np.log1p(rest)
            ent[r] = np.log1p(rest) - np.where(e > 0, e * np.where(e > 0, d, 0), 0).sum() / (1 + rest)
        t = tokens[r]
        lp[r] = 0.0 if t < 0 else np.nan if t >= V else logp[t]
        top[r] = logp[order[r]]
    return lp, ent, order, top


def run_logprobs(raw, t, V, tokens, n_top, T, offset=0):
    """raw [rows][stride] activations; `offset` elements before the first row."""
    rows, stride = raw.shape
    buf = put(np.concatenate([np.zeros(offset, raw.dtype), raw.reshape(-1)]))
    ws = K.DeviceBuffer(K.token_logprobs_workspace(rows, V))
    ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))
    o = [K.DeviceBuffer(4 * rows) for _ in range(2)] + [K.DeviceBuffer(max(4, 4 * rows * n_top)) for _ in range(2)]
    K.token_logprobs(t, buf.ptr + offset * raw.itemsize, rows, V, ws, tokens=i32(tokens), logprob=o[0], entropy=o[1], n_top=n_top,
                     top_idx=o[2] if n_top else None, top_logprob=o[3] if n_top else None, temperature=T, row_stride=stride)
    return (o[0].download(np.float32, rows), o[1].download(np.float32, rows),
            o[2].download(np.int32, rows * n_top).reshape(rows, n_top), o[3].download(np.float32, rows * n_top).reshape(rows, n_top))


def check_logprobs(x, raw, t, tokens, n_top, T, offset=0):
    """Sums of f32 terms: a term is off by 4 U (its exponent's argument in two parts, the
    exponential) and, of d binades below 1, by d U more; chains of 32 additions, then
    pairwise.  48 U of the sum covers them, as an absolute error of its logarithm; an
    entropy's terms weigh d (at most 40 before they vanish) more."""
    V = x.shape[1]
    got = run_logprobs(raw, t, V, tokens, n_top, T, offset)
    want = logprobs64(x, tokens, n_top, T)
    with np.errstate(invalid="ignore"):
        # relative to the sum without the largest term: a likely token's log probability keeps its digits
        small = lambda w: 48 * U * np.minimum(1.0, np.abs(w)) + 2 * U * np.abs(w) + 1e-37
        close(got[0], want[0], small(want[0]), "logprob")
        close(got[1], want[1], 48 * U * np.minimum(40.0, 40.0 * np.abs(want[1])) + 2 * U * np.abs(want[1]) + 1e-37, "entropy")
        assert np.array_equal(got[2], want[2])
        close(got[3], want[3], small(want[3]), "top")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V,pad,rows,n_top,T", [
    (1, 0, 1, 1, 1.0), (2, 0, 3, 2, 1.0), (5, 1, 2, 5, 0.7), (63, 0, 5, 20, 1.0), (64, 1, 2, 32, 2.0), (2047, 0, 3, 1, 1.0),
    (2048, 3, 4, 20, 0.5), (2049, 0, 3, 32, 1.0), (4097, 1, 9, 3, 1.3), (50257, 0, 3, 20, 1.0), (151936, 0, 2, 5, 0.8),
    (70000, 7, 1, 0, 1.0), (1 << 20, 0, 1, 32, 1.0)])
def test_token_logprobs(device, t, V, pad, rows, n_top, T):
    print(f"logprobs type {t} vocab {V} rows {rows} top {n_top} T {T}", flush=True)
    rng = np.random.default_rng([V, rows, n_top, t])
    x = 3 * rng.normal(size=(rows, V + pad))
    x[:, V:] = 1e4  # past the vocabulary: not read
    x[0, rng.integers(0, V)] += 12
    raw = encode(x, t)
    tokens = rng.integers(0, V, rows)
    tokens[0] = int(np.argmax(x[0, :V]))
    for offset in (0, 1):
        check_logprobs(decode(raw, t)[:, :V], raw, t, tokens, n_top, T, offset)


@pytest.mark.parametrize("t", TYPES)
def test_token_logprobs_ties_and_masks(device, t):
    """Ties go to the lowest index, +0 and -0 tie; -inf and the type's lowest value rule
    tokens out; rows with nothing left, one token left, a NaN, +inf; tokens out of range."""
    V, n_top = 5000, 32
    rng = np.random.default_rng(t)
    low = {F32: -3.4028234663852886e38, F16: -65504.0, BF16: -3.3895313892515355e38}[t]
    rows = []
    rows.append(np.zeros(V))                                      # all alike
    r = np.zeros(V); r[::2] = -0.0; rows.append(r)
    rows.append(np.full(V, -np.inf))                              # nothing left
    r = np.full(V, -np.inf); r[4321] = 2.5; rows.append(r)        # one left
    r = np.full(V, low); r[[17, 3000]] = [1.0, 1.0]; rows.append(r)
    rows.append(np.full(V, low))                                  # all at the lowest value
    r = np.full(V, -np.inf); r[rng.permutation(V)[:20]] = rng.integers(0, 3, 20); rows.append(r)
    r = rng.normal(size=V); r[2049] = np.nan; rows.append(r)
    r = rng.normal(size=V); r[77] = np.inf; rows.append(r)
    rows.append(np.sort(rng.integers(0, 50, V)).astype(float))    # the largest all in the last piece
    rows.append(np.sort(rng.integers(0, 50, V))[::-1].astype(float))
    r = rng.normal(size=V); r[10] = 40.0; rows.append(r)          # one token nearly certain
    raw = encode(np.stack(rows), t)
    x = decode(raw, t)
    tokens = rng.integers(0, V, len(rows))
    tokens[:4] = [-1, V, 5, 4321]
    tokens[4], tokens[6], tokens[11] = 3000, 0, 10
    check_logprobs(x, raw, t, tokens, n_top, 1.0)
    tokens[:3] = [-2 ** 31, 2 ** 31 - 1, V - 1]
    check_logprobs(x, raw, t, tokens, 1, 0.6)


@pytest.mark.parametrize("t,V,rows,n_top", [(F32, 5000, 131, 32), (BF16, 3000, 300, 7), (F16, 600000, 129, 20),
                                            (F32, 5000, 257, 32), (F16, 600000, 259, 20)])
def test_token_logprobs_many_rows(device, t, V, rows, n_top):
    """Rows enough for the narrower join, more pieces than it has threads among them;
    the rows repeat a few of their own, so that ties and sorted rows come along."""
    print(f"logprobs type {t} vocab {V} rows {rows} top {n_top}", flush=True)
    rng = np.random.default_rng([V, rows])
    kinds = np.stack([3 * rng.normal(size=V), np.sort(rng.integers(0, 50, V)).astype(float), np.zeros(V),
                      np.where(rng.random(V) < 0.99, -np.inf, rng.normal(size=V))])
    raw4 = encode(kinds, t)
    pick = rng.integers(0, 4, rows)
    tokens4 = rng.integers(0, V, 4)
    want = logprobs64(decode(raw4, t), tokens4, n_top, 1.0)
    got = run_logprobs(raw4[pick], t, V, tokens4[pick], n_top, 1.0)
    with np.errstate(invalid="ignore"):
        for g, w, what, d in ((got[0], want[0], "logprob", 1.0), (got[1], want[1], "entropy", 40.0), (got[3], want[3], "top", 1.0)):
            close(g, w[pick], 48 * U * np.minimum(d, d * np.abs(w[pick])) + 2 * U * np.abs(w[pick]) + 1e-37, what)
    assert np.array_equal(got[2], want[2][pick])


def test_token_logprobs_parts(device):
    """Each output alone, and nothing else written."""
    rng = np.random.default_rng(0)
    x = rng.normal(size=(3, 3000)).astype(np.float32)
    buf, ws = put(x), K.DeviceBuffer(K.token_logprobs_workspace(3, 3000))
    lp, ent = K.DeviceBuffer(12), K.DeviceBuffer(12)
    want = logprobs64(x.astype(np.float64), [1, 2, 3], 1, 1.0)
    K.token_logprobs(F32, buf, 3, 3000, ws, tokens=i32([1, 2, 3]), logprob=lp)
    close(lp.download(np.float32, 3), want[0], 48 * U + 2 * U * np.abs(want[0]), "logprob")
    K.token_logprobs(F32, buf, 3, 3000, ws, entropy=ent)
    close(ent.download(np.float32, 3), want[1], 48 * 40 * U, "entropy")
    K.token_logprobs(F32, buf, 3, 3000, ws)  # nothing asked for
    K.token_logprobs(F32, buf, 0, 3000, ws, entropy=ent)


# ------------------------------------------------------------------ together

class Step:
    """One speculative step on buffers of its own: rotary positions, rows stored, the
    drafts' attention, log probabilities of stand-in logits, the accepted path moved."""

    def __init__(self, fmt, rng, stream=None, n=2, T=6, ctx=220):
        self.fmt, self.stream, self.n, self.T, self.ctx = fmt, stream, n, T, ctx
        self.nh, self.nk, self.D, self.V = 8, 2, 128, 3001
        row = (self.nh + 2 * self.nk) * self.D
        self.cache = K.KvCache.allocate(fmt, n, self.nk, ctx, self.D)
        self.old = fill_cache(self.cache, rng)
        self.prefix = np.array([150, 97][:n])
        self.x = rng.normal(size=(n * T, row)).astype(np.float32)
        self.sees = np.stack([tree_bits(rng, T) for _ in range(n)])
        self.depth = self.sees.sum(-1) - 1
        self.inv, _ = K.rope_freqs(self.D, 1e6)
        self.w = [(1 + 0.1 * rng.normal(size=self.D)).astype(np.float32) for _ in range(2)]
        self.logits = (3 * rng.normal(size=(n * T, self.V))).astype(np.float32)
        self.tokens = rng.integers(0, self.V, n * T)
        self.path = np.array([[0, 2, 4], [0, 1, 5]][:n])
        d = self.d = {}
        d["x"], d["pos"] = put(self.x), i32((self.prefix[:, None] + self.depth).reshape(-1))
        d["inv"], d["wq"], d["wk"] = put(self.inv), put(self.w[0]), put(self.w[1])
        d["prefix"], d["mask"] = i32(self.prefix), put(mask_words(self.sees))
        d["logits"], d["tokens"] = put(self.logits), i32(self.tokens)
        d["path"] = i32(self.prefix[:, None] + self.path)
        d["q"], d["k"] = K.DeviceBuffer(4 * n * T * self.nh * self.D), K.DeviceBuffer(4 * n * T * self.nk * self.D)
        d["out"] = K.DeviceBuffer(4 * n * T * self.nh * self.D)
        d["ws"] = K.DeviceBuffer(K.attention_tree_workspace(self.cache, self.nh, T, 160))
        d["lws"] = K.DeviceBuffer(K.token_logprobs_workspace(n * T, self.V))
        for m, e in (("lp", 1), ("ent", 1), ("top", 4), ("top_lp", 4)):
            d[m] = K.DeviceBuffer(4 * n * T * e)
        d["pk"], d["pv"] = (K.DeviceBuffer(4 * n * 3 * self.nk * self.D) for _ in range(2))

    def verify(self):
        d, n, T, s = self.d, self.n, self.T, self.stream
        row, nh, nk, D = self.x.shape[1], self.nh, self.nk, self.D
        K.rope(F32, d["x"].ptr, d["x"].ptr + 4 * nh * D, d["pos"], d["inv"], n * T, nh, nk, D, q_out=d["q"], k_out=d["k"],
               q_norm=d["wq"], k_norm=d["wk"], q_stride=row, k_stride=row, stream=s)
        # keys from the rotated rows, values from the projections: two strides, so packed rows of each
        K.check(K.lib().knj_kv_store(self.cache.ref, F32, d["k"].ptr, self.values_ptr(), nk * D, d["prefix"].ptr, None, T, s))
        K.attention_tree(self.cache, F32, d["q"], d["out"], nh, T, d["prefix"], 160, d["ws"], mask=d["mask"], stream=s)
        K.token_logprobs(F32, d["logits"], n * T, self.V, d["lws"], tokens=d["tokens"], logprob=d["lp"], entropy=d["ent"],
                         n_top=4, top_idx=d["top"], top_logprob=d["top_lp"], stream=s)

    def values_ptr(self):
        if "v" not in self.d:
            v = self.x[:, (self.nh + self.nk) * self.D:]
            self.d["v"] = put(np.ascontiguousarray(v))
        return self.d["v"].ptr

    def accept(self):
        K.kv_load(self.cache, F32, self.d["pk"], self.d["pv"], 3, slots=self.d["path"], stream=self.stream)
        K.kv_store(self.cache, F32, self.d["pk"], self.d["pv"], self.d["prefix"], 3, stream=self.stream)

    def outputs(self):
        d, r = self.d, self.n * self.T
        return [d["out"].download(np.float32), d["lp"].download(np.float32, r), d["ent"].download(np.float32, r),
                d["top"].download(np.int32, 4 * r), d["top_lp"].download(np.float32, 4 * r)]


@pytest.mark.parametrize("fmt", FORMATS)
def test_speculative_step(device, fmt):
    """The whole step against float64 from the projections on, each stage given what
    the stage before it wrote where that is a rounding (the cache's codes)."""
    rng = np.random.default_rng(fmt)
    st = Step(fmt, rng)
    st.verify()
    K.synchronize()
    n, T, nh, nk, D = st.n, st.T, st.nh, st.nk, st.D
    x = st.x.astype(np.float64).reshape(n * T, nh + 2 * nk, D)
    pos = (st.prefix[:, None] + st.depth).reshape(-1)
    w = [a.astype(np.float64) for a in st.w]
    q = rope64(x[:, :nh], w[0], pos, st.inv, 1.0, D, K.ROPE_HALF, 1e-6)
    k = rope64(x[:, nh:nh + nk], w[1], pos, st.inv, 1.0, D, K.ROPE_HALF, 1e-6)
    a = cache_arrays(st.cache)
    kv = [values(a[m], a[m + "_scale"], fmt) for m in ("k", "v")]
    # the drafts' rows in the cache: within a step of the format of the row's largest
    step = {K.KV_F16: 2.0 ** -11, K.KV_I8: 0.51 / 127, K.KV_F8: 2.0 ** -4 * 1.01}[fmt]
    for m, rows in ((0, k), (1, x[:, nh + nk:])):
        r = rows.reshape(n, T, nk, D)
        for s in range(n):
            got = kv[m][s, :, st.prefix[s]:st.prefix[s] + T].transpose(1, 0, 2)
            big = np.abs(r[s]).max(-1, keepdims=True)
            close(got, r[s], step * big * 1.001, "stored")
            others = np.ones(st.ctx, bool)
            others[st.prefix[s]:st.prefix[s] + T] = False
            assert np.array_equal(kv[m][s][:, others], st.old[m][s][:, others])
    got = st.outputs()
    # the rotated queries come with the rope's own error (24 U of a head's largest)
    want, bound = tree64(q.reshape(n, T, nh, D), kv, st.prefix, [T] * n, st.sees, D ** -0.5, F32)
    extra = 2 * 24 * U * np.abs(q).max() * max(np.abs(kv[0][s]).sum(-1).max() for s in range(n)) * D ** -0.5
    close(got[0].reshape(n, T, nh, D), want, bound + extra * np.abs(kv[1]).max(), "attention")
    lw = logprobs64(st.logits.astype(np.float64), st.tokens, 4, 1.0)
    close(got[1], lw[0], 50 * U + 2 * U * np.abs(lw[0]), "logprob")
    assert np.array_equal(got[3].reshape(-1, 4), lw[2])
    # the accepted path moves to the end of the prefix with its codes
    st.accept()
    b = cache_arrays(st.cache)
    for m in ("k", "v"):
        for s in range(n):
            assert np.array_equal(b[m][s][:, st.prefix[s]:st.prefix[s] + 3], a[m][s][:, st.prefix[s] + st.path[s]])


def test_step_matches_attention_step(device):
    """A chain verified over the model's own cache layout gives what the decode step
    gives token by token: attention_step forms its angles in f32 (off by pos * 2^-24)
    and rounds its own rotated key to f16, so a key part by one f16 step at most."""
    rng = np.random.default_rng(3)
    nh, nk, D, T, P, ctx = 32, 4, 128, 3, 90, 128
    c = K.KvCache.allocate(K.KV_F16, 1, nk, ctx, D)
    fill_cache(c, rng, 0.0)
    c2 = K.KvCache.allocate(K.KV_F16, 1, nk, ctx, D)
    for m in ("k", "v"):
        getattr(c2, m).upload(getattr(c, m).download(np.uint16))
    x = rng.normal(size=(T, (nh + 2 * nk) * D)).astype(np.float32)
    w = [put((1 + 0.1 * rng.normal(size=D)).astype(np.float32)) for _ in range(2)]
    dx = put(x)
    step = []
    for t in range(T):
        at = dx.ptr + 4 * t * x.shape[1]
        o = K.DeviceBuffer(4 * nh * D)
        K.attention_step(at, at + 4 * nh * D, at + 4 * (nh + nk) * D, w[0], w[1], 1e-6, 1e6, P + t, nh, nk, D, ctx, c.k, c.v, o)
        step.append(o.download(np.float32))
    inv, _ = K.rope_freqs(D, 1e6)
    q, k = K.DeviceBuffer(4 * T * nh * D), K.DeviceBuffer(4 * T * nk * D)
    row = x.shape[1]
    K.rope(F32, dx.ptr, dx.ptr + 4 * nh * D, i32(P + np.arange(T)), put(inv), T, nh, nk, D, q_out=q, k_out=k, q_norm=w[0],
           k_norm=w[1], q_stride=row, k_stride=row)
    v = put(np.ascontiguousarray(x[:, (nh + nk) * D:]))
    K.kv_store(c2, F32, k, v, i32([P]), T)
    out = K.DeviceBuffer(4 * T * nh * D)
    ws = K.DeviceBuffer(K.attention_tree_workspace(c2, nh, T, P))
    K.attention_tree(c2, F32, q, out, nh, T, i32([P]), P, ws)
    a, b = cache_arrays(c), cache_arrays(c2)
    assert np.array_equal(a["v"], b["v"])
    ka, kb = (z["k"].view(np.float16).astype(np.float64) for z in (a, b))
    # an f16 step of the larger of a pair (a rotation moves parts between the two)
    close(kb, ka, 2.0 ** -10 * np.maximum(np.abs(ka), 1e-2) + 2.0 ** -16, "keys")
    # scores part by the angles' and the key's difference: 2^-24 * 93 * |q||k| + 2^-10 * a few elements
    close(out.download(np.float32).reshape(T, -1), np.stack(step), 2e-4 * np.abs(np.stack(step)).max(), "attention")


def hip():
    """The HIP runtime the library itself is linked against."""
    h = C.CDLL("libamdhip64.so")
    P = C.c_void_p
    for name, args in [("hipStreamCreateWithFlags", [C.POINTER(P), C.c_uint]), ("hipStreamDestroy", [P]),
                       ("hipStreamBeginCapture", [P, C.c_int]), ("hipStreamEndCapture", [P, C.POINTER(P)]),
                       ("hipGraphInstantiate", [C.POINTER(P), P, P, P, C.c_size_t]), ("hipGraphLaunch", [P, P]),
                       ("hipGraphExecDestroy", [P]), ("hipGraphDestroy", [P]), ("hipGetDeviceCount", [C.POINTER(C.c_int)]),
                       ("hipSetDevice", [C.c_int])]:
        getattr(h, name).argtypes = args
        getattr(h, name).restype = C.c_int
    return h


@pytest.fixture
def streams(device):
    """Two streams that do not wait for the default one."""
    h, s = hip(), [C.c_void_p() for _ in range(2)]
    for z in s:
        assert h.hipStreamCreateWithFlags(C.byref(z), 1) == 0
    yield s
    K.synchronize()
    for z in s:
        h.hipStreamDestroy(z)


def test_two_streams_at_once(streams):
    """Two steps on two streams, a workspace each, give what each gives alone."""
    steps = [Step(f, np.random.default_rng(f), stream=z) for f, z in ((K.KV_I8, streams[0]), (K.KV_F8, streams[1]))]
    for st in steps:
        st.values_ptr()
    K.synchronize()
    want = []
    for st in steps:
        st.verify()
        K.synchronize()
        want.append(st.outputs())
        st.d["out"].zero()
    K.synchronize()
    for _ in range(10):
        for st in steps:
            st.verify()
    K.synchronize()
    for st, w in zip(steps, want):
        for a, b in zip(st.outputs(), w):
            assert np.array_equal(a, b)


def test_step_in_graphs(streams):
    """Captured steps: replayed several times with inputs changed in between, with eager
    work and synchronisation between replays; two graphs with a workspace each."""
    h, stream = hip(), streams[0]
    steps = [Step(f, np.random.default_rng(f), stream=stream) for f in (K.KV_I8, K.KV_F16)]
    graphs = []
    for st in steps:
        st.values_ptr()
        st.verify()
        K.synchronize()
        graph, exe = C.c_void_p(), C.c_void_p()
        assert h.hipStreamBeginCapture(stream, 2) == 0  # hipStreamCaptureModeRelaxed
        st.verify()
        assert h.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert h.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
        graphs.append((graph, exe))
    rng = np.random.default_rng(9)
    for _ in range(4):
        for st, (_, exe) in zip(steps, graphs):
            st.d["prefix"].upload(rng.integers(20, 160, st.n).astype(np.int32))
            st.d["x"].upload(rng.normal(size=st.x.shape).astype(np.float32))
            st.d["logits"].upload(rng.normal(size=st.logits.shape).astype(np.float32))
            for m in ("out", "lp", "ent", "top", "top_lp"):
                st.d[m].zero()
            K.synchronize()
            assert h.hipGraphLaunch(exe, stream) == 0
            K.synchronize()
            got = st.outputs()
            for m in ("out", "lp", "ent", "top", "top_lp"):
                st.d[m].zero()
            K.synchronize()
            st.verify()  # eager, on the same inputs (the cache rows are the same rows again)
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
    c = K.KvCache.allocate(K.KV_F16, 1, 1, 8, 64)
    buf = K.DeviceBuffer(4096)
    assert h.hipSetDevice(1) == 0
    try:
        with pytest.raises(K.KnjError) as e:
            K.kv_load(c, F32, buf, buf, 1)
        assert e.value.code == K.KNJ_E_STATE
    finally:
        assert h.hipSetDevice(0) == 0
