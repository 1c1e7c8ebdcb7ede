"""GPU: the speculative-step operators at the ends of their ranges -- bits of the
softmax's weights, outliers among value scales, rows that are not drafts,
queries and cache rows of extreme units, angles and norms of rotations, small
vocabularies -- against float64."""
import numpy as np
import pytest

import kanjoos_amd as K
import test_gpu_spec as S

pytestmark = pytest.mark.gpu

F32, F16, BF16 = S.F32, S.F16, S.BF16
U, HALF, TYPES, FORMATS = S.U, S.HALF, S.TYPES, S.FORMATS


# (query heads of the one kv head, drafts, bound on the prefix): tiles of 16, 32, 64 and 128 columns
TILES = [(4, 3, 300), (8, 4, 300), (16, 4, 640000), (16, 8, 640000)]


@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nh,T,bound_p", TILES)
def test_weights_keep_their_bits(device, t, fmt, D, nh, T, bound_p):
    """16-bit activations: the softmax's weights round no earlier than with f32 ones.
    Values in pairs v, -v under nearly equal weights leave little of an output, so that
    its own rounding hides nothing: weights of 11 bits would be 2^-12 of a value off."""
    print(f"weights type {t} format {fmt} D {D} heads {nh} drafts {T}", flush=True)
    rng = np.random.default_rng([t, fmt, D, nh, T])
    P = 130
    c = K.KvCache.allocate(fmt, 1, 1, bound_p + T, D)
    k, v = rng.normal(size=(2, 1, P + T, 1, D))
    v[:, 1::2] = -v[:, 0:-1:2]
    kv = S.store_prefix(c, [0.1 * k, v], P + T)
    q = S.decode(S.encode(0.1 * rng.normal(size=(1, T, nh, D)), t), t)
    sees = np.eye(T, dtype=bool)[None]
    got, _ = S.run_tree(c, t, q, T, [P], None, sees, nh, max_prefix=bound_p)
    want, bound = S.tree64(q, kv, [P], [T], sees, D ** -0.5, F32)
    assert np.abs(want).mean() < 0.1 * np.abs(v).mean()
    S.close(got, want, bound + HALF[t] * np.abs(want) + (2.0 ** -25 if t == F16 else 0.0), "weights")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("nh,T", [(16, 2), (32, 4), (64, 12)])
def test_rows_that_are_not_drafts(device, t, fmt, nh, T):
    """What the queries of rows past the counts, or of another draft, hold -- NaN,
    infinities, large values -- changes no bit of a draft's output, over prefixes of
    many chunks and scores that keep growing."""
    print(f"other rows type {t} format {fmt} heads {nh} drafts {T}", flush=True)
    rng = np.random.default_rng([t, fmt, nh, T])
    n, nk, D, P = 8, 8, 64, 3000
    c = S.make_cache(fmt, n, nk, P + T, D)
    ramp = np.linspace(0, 1, P + T)[None, :, None, None]
    base = rng.normal(size=(nk, D))
    kv = S.store_prefix(c, [rng.normal(size=(n, P + T, nk, D)) + 2 * ramp * base, rng.normal(size=(n, P + T, nk, D))], P + T)
    sees = np.stack([S.tree_bits(rng, T) for _ in range(n)])
    prefixes = P - 100 * np.arange(n)
    counts = np.array([T - 1] * n)
    q = 1.5 * np.repeat(base, nh // nk, axis=0) + rng.normal(size=(n, T, nh, D))
    q = S.decode(S.encode(q, t), t)
    clean, _ = S.run_tree(c, t, q, T, prefixes, counts, sees, nh)
    want, bound = S.tree64(q[:2], [a[:2] for a in kv], prefixes[:2], counts[:2], sees[:2], D ** -0.5, F32)
    S.close(clean[:2, :T - 1], want[:, :T - 1], (bound + HALF[t] * np.abs(want) + 2.0 ** -25)[:, :T - 1], "clean")
    for what in (np.nan, np.inf, -np.inf, 1e4):
        other = q.copy()
        other[:, T - 1] = what * np.sign(rng.normal(size=other[:, T - 1].shape))
        with np.errstate(invalid="ignore"):
            got, _ = S.run_tree(c, t, other, T, prefixes, counts, sees, nh)
        assert np.array_equal(got[:, :T - 1], clean[:, :T - 1]), what
        if T > 2:  # a draft among the others
            other = q.copy()
            other[:, 1, ::3] = what
            with np.errstate(invalid="ignore"):
                got, _ = S.run_tree(c, t, other, T, prefixes, counts, sees, nh)
            assert np.array_equal(got[:, [0, 2]], clean[:, [0, 2]]), what


def tree64p(q, kv, amax, prefix, sees, scale, t):
    """Attention of full sets of drafts in float64, with a bound that weighs each slot's
    error by its own share: a weight is off by 32 U |q||k| scale + 64 U of itself, and
    by 2^-25 of the largest product of a share p and its row's largest magnitude
    (`amax`), at random over the slots: six standard deviations."""
    n, T, nh, D = q.shape
    nk = kv[0].shape[1]
    out, bound = np.empty(q.shape), np.empty(q.shape)
    for s in range(n):
        for h in range(nh):
            kh = h * nk // nh
            for i in range(T):
                slots = np.concatenate([np.arange(prefix[s]), prefix[s] + np.nonzero(sees[s, i])[0]]).astype(int)
                ks, vs = kv[0][s, kh][slots], kv[1][s, kh][slots]
                x = scale * (ks @ q[s, i, h])
                p = np.exp(x - x.max())
                p /= p.sum()
                o = p @ vs
                off = p * (32 * U * scale * (np.abs(ks) @ np.abs(q[s, i, h])) + 64 * U)
                out[s, i, h] = o
                bound[s, i, h] = off @ np.abs(vs) + off.sum() * np.abs(o) + 6 * 2.0 ** -25 * np.sqrt(slots.size) * (p * amax[s, kh][slots]).max() \
                    + HALF[t] * np.abs(o) + (2.0 ** -25 if t == F16 else 2.0 ** -126)
    return out, bound


def steered(rng, q, nk, P, nats, sizes, noise=0.3):
    """Keys and values [1][P][nk][D] of P slots whose scores against every row of q are about
    `nats` (before the 1/sqrt(D) is taken out) and whose values are about `sizes`."""
    D = q.shape[-1]
    u = q.mean((0, 1)).reshape(nk, -1, D).mean(1)
    u /= (u * u).sum(-1, keepdims=True)
    k = D ** 0.5 * np.asarray(nats)[None, :, None, None] * u + noise * rng.normal(size=(1, P, nk, D))
    return k, rng.normal(size=(1, P, nk, D)) * np.asarray(sizes)[None, :, None, None]


LN2 = float(np.log(2.0))
# per slot of P: scores in nats and sizes of the values
UNITS = {
    "one slot of 2^16": lambda P, at: (np.where(np.arange(P) == at, -30.0, 0.0), np.where(np.arange(P) == at, 2.0 ** 16, 1.0)),
    "one slot of 2^28": lambda P, at: (np.where(np.arange(P) == at, -40.0, 0.0), np.where(np.arange(P) == at, 2.0 ** 28, 1.0)),
    "one slot of 2^40": lambda P, at: (np.where(np.arange(P) == at, -60.0, 0.0), np.where(np.arange(P) == at, 2.0 ** 40, 1.0)),
    "one slot of 2^40, no weight": lambda P, at: (np.where(np.arange(P) == at, -300.0, 0.0), np.where(np.arange(P) == at, 2.0 ** 40, 1.0)),
    "one heavy slot of 2^-30": lambda P, at: (np.where(np.arange(P) == at, 24.0, 0.0), np.where(np.arange(P) == at, 2.0 ** -30, 1.0)),
    "shares and sizes opposed": lambda P, at: (-40 * LN2 * np.arange(P) / P, 2.0 ** (40 * np.arange(P) / P)),
    "sizes fall twice as fast": lambda P, at: (20 * LN2 * np.arange(P) / P, 2.0 ** (-40 * np.arange(P) / P)),
    "sizes fall, scores rise": lambda P, at: (40 * LN2 * np.arange(P) / P, 2.0 ** (-20 * np.arange(P) / P)),
    "heavy tails": lambda P, at: tuple(f(np.random.default_rng(5).normal(size=(2, P))[i]) for i, f in enumerate((lambda z: 8 * z, lambda z: 2.0 ** (8 * z)))),
    "waves": lambda P, at: (20 * np.sin(np.arange(P) / 40), 2.0 ** (20 * np.cos(np.arange(P) / 70))),
}


@pytest.mark.parametrize("fmt", [K.KV_F8, K.KV_I8])
@pytest.mark.parametrize("tile", range(len(TILES)))
@pytest.mark.parametrize("units", list(UNITS))
def test_units_of_values(device, fmt, tile, units):
    """8-bit values whose scales lie far apart: what an output is made of keeps its bits
    whatever slots of next to no weight hold, wherever they lie (the activations' types
    in turn)."""
    t, (nh, T, bound_p) = TYPES[(list(UNITS).index(units) + fmt + tile) % 3], TILES[tile]
    print(f"units '{units}' type {t} format {fmt} heads {nh} drafts {T}", flush=True)
    rng = np.random.default_rng([t, fmt, nh, T])
    D, P = 64, 900
    c = K.KvCache.allocate(fmt, 1, 1, max(bound_p, P) + T, D)
    q = S.decode(S.encode(2 * rng.normal(size=D) + 0.1 * rng.normal(size=(1, T, nh, D)), t), t)
    sees = S.tree_bits(rng, T)[None]
    for at in (3, 200, 700, P - 1, P + T - 1) if "slot" in units else (0,):
        nats, sizes = UNITS[units](P + T, at)
        k, v = steered(rng, q, 1, P + T, nats, sizes)
        kv = S.store_prefix(c, [k, v], P + T)
        amax = np.abs(v).max(-1).transpose(0, 2, 1)
        with np.errstate(over="ignore"):
            got, _ = S.run_tree(c, t, q, T, [P], None, sees, nh, max_prefix=max(bound_p, P))
            want, bound = tree64p(q, kv, amax, [P], sees, D ** -0.5, t)
        if t == F16:
            assert np.abs(want).max() < 65000
        S.close(got, want, bound, f"outlier at {at}")
        # the bits of a draft hang on nothing that its neighbours hold
        if T > 3:
            other = q.copy()
            other[:, T - 1] = np.nan
            with np.errstate(invalid="ignore"):
                again, _ = S.run_tree(c, t, other, T, [P], None, sees, nh, max_prefix=max(bound_p, P))
            assert np.array_equal(again[:, :T - 1], got[:, :T - 1])


@pytest.mark.parametrize("fmt", [K.KV_F8, K.KV_I8])
@pytest.mark.parametrize("nh,T,t", [(4, 3, F32), (16, 6, BF16)])
@pytest.mark.parametrize("units", list(UNITS))
def test_units_over_splits(device, fmt, nh, T, t, units):
    """The same over sequences whose slots are split over workgroups of many chunks each."""
    print(f"units '{units}' over splits type {t} format {fmt} heads {nh} drafts {T}", flush=True)
    rng = np.random.default_rng([fmt, nh, T])
    n, nk, D, P = 32, 2, 64, 2000
    c = K.KvCache.allocate(fmt, n, nk, P + T, D)
    q = S.decode(S.encode(2 * rng.normal(size=D) + 0.1 * rng.normal(size=(n, T, nh, D)), t), t)
    nats, sizes = UNITS[units](P + T, 1234)
    parts = [steered(rng, q[s:s + 1], nk, P + T, nats, sizes) for s in range(n)]
    k, v = (np.concatenate([p[i] for p in parts]) for i in range(2))
    kv = S.store_prefix(c, [k, v], P + T)
    sees = np.stack([S.tree_bits(rng, T)] * n)
    got, _ = S.run_tree(c, t, q, T, [P] * n, None, sees, nh)
    assert np.isfinite(got).all()
    some = [0, 13, 31]
    want, bound = tree64p(q[some], [a[some] for a in kv], np.abs(v).max(-1).transpose(0, 2, 1)[some], [P] * 3, sees[some], D ** -0.5, t)
    S.close(got[some], want, bound, "split")


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("fmt,size", [(f, z) for f in FORMATS for z in (-140, -112, -101, 30, 112, 117, 126) if f != K.KV_F16 or z <= 30])
@pytest.mark.parametrize("nh,T,bound_p", TILES)
def test_queries_of_any_size(device, t, fmt, nh, T, bound_p, size):
    """Queries up to the ends of f32's range, 2^size, against keys and a scale that keep
    the scores ordinary (of the smallest: next to nothing, every slot the same; no f16
    keys suit the largest)."""
    ksize = 2.0 ** (-10 if size > 0 else 0) if fmt == K.KV_F16 else 2.0 ** min(95, max(-114, -size))
    scale = float(np.float32(min(1e6, max(1e-6, 2.0 ** -size / ksize / 8))))
    print(f"queries of 2^{size} type {t} format {fmt} heads {nh} drafts {T}", flush=True)
    rng = np.random.default_rng([t, fmt, nh, T, size + 200])
    D, P = 64, 300
    c = K.KvCache.allocate(fmt, 1, 1, max(bound_p, P) + T, D)
    k, v = rng.normal(size=(2, 1, P + T, 1, D))
    kv = S.store_prefix(c, [ksize * k, v], P + T)
    q = S.decode(S.encode(np.clip(rng.normal(size=(1, T, nh, D)), -3.9, 3.9) * 2.0 ** size, t), t)
    assert np.isfinite(q).all()
    sees = S.tree_bits(rng, T)[None]
    got, _ = S.run_tree(c, t, q, T, [P], None, sees, nh, max_prefix=max(bound_p, P), scale=scale)
    want, bound = S.tree64(q, kv, [P], [T], sees, scale, F32)
    S.close(got, want, bound + HALF[t] * np.abs(want), "queries")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("nh,T,bound_p", TILES)
def test_largest_scores(device, t, fmt, nh, T, bound_p):
    """Scores to 2^25, far from one another: the largest slot's value row is the output."""
    rng = np.random.default_rng([t, fmt, nh, T])
    D, P = 64, 700
    c = K.KvCache.allocate(fmt, 1, 1, max(bound_p, P) + T, D)
    k, v = rng.normal(size=(2, 1, P + T, 1, D))
    kv = S.store_prefix(c, [1000 * k, v], P + T)
    q = S.decode(S.encode(700 * rng.normal(size=(1, T, nh, D)), t), t)
    sees = np.eye(T, dtype=bool)[None]
    got, _ = S.run_tree(c, t, q, T, [P], None, sees, nh, max_prefix=max(bound_p, P), scale=1.0)
    for i in range(T):
        slots = np.append(np.arange(P), P + i)
        sc = q[0, i] @ kv[0][0, 0][slots].T
        order = np.sort(sc, axis=-1)
        assert 2.0 ** 22 < np.abs(sc).max() < 2.0 ** 25
        clear = order[:, -1] - order[:, -2] > 300  # (a score is off by 2^-20 of |q||k|, 2^27)
        want = kv[1][0, 0][slots[sc.argmax(-1)]]
        # of the one weight: times its scale U, as two parts of 11 bits 2 U, their products' sum U, joined with
        # other splits' zeros 2 U, over the sum of weights 2 U; then the output's rounding
        S.close(got[0, i][clear], want[clear], (8 * U + HALF[t]) * np.abs(want[clear]) + (2.0 ** -25 if t == F16 else 0.0), "largest")
        assert clear.any()


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("fmt", [K.KV_F8, K.KV_I8])
@pytest.mark.parametrize("nh,T,bound_p", TILES + [(4, 3, 12000)])
@pytest.mark.parametrize("low,high", [(-118.95, -117.3), (-119.0, -110.0), (90.0, 100.0), (119.0, 127.9), (-118.9, 127.9)])
def test_values_of_any_size(device, t, fmt, nh, T, bound_p, low, high):
    """8-bit value rows whose largest magnitudes lie between 2^low and 2^high, to both
    ends of what a cache holds (e4m3 scales below f32's normal numbers among them)."""
    print(f"values of 2^{low} to 2^{high} type {t} format {fmt} heads {nh} drafts {T}", flush=True)
    rng = np.random.default_rng([t, fmt, nh, T, int(low) + 200])
    D, P = 64, 300
    c = K.KvCache.allocate(fmt, 1, 1, max(bound_p, P) + T, D)
    k, v = rng.normal(size=(2, 1, P + T, 1, D))
    v *= 2.0 ** rng.uniform(low, high, size=(1, P + T, 1, 1)) / np.abs(v).max(-1, keepdims=True)
    v[:, 7::40] = 0
    kv = S.store_prefix(c, [k, v], P + T)
    assert np.all(np.abs(kv[1]).max(-1)[..., [0, 100, P]] > 0)
    q = S.decode(S.encode(rng.normal(size=(1, T, nh, D)), t), t)
    sees = S.tree_bits(rng, T)[None]
    got, _ = S.run_tree(c, t, q, T, [P], None, sees, nh, max_prefix=max(bound_p, P))
    want, bound = S.tree64(q, kv, [P], [T], sees, D ** -0.5, F32)
    S.close(got, want, bound - 1e-37 + HALF[t] * np.abs(want) + 2.0 ** (-148 if t == F32 else -134), "values")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V,n_top", [(33, 32), (300, 2), (300, 32), (2048, 20), (2049, 3), (4097, 4), (8000, 20), (32000, 17), (32000, 32),
                                     (2048 * 19 - 5, 20)])
def test_largest_of_small_vocabularies(device, t, V, n_top):
    """Fewer pieces of 2048 logits than alternatives asked for: rows in any order, with
    ties across the threshold, with few or no tokens left, with NaN; few rows and many."""
    print(f"small vocabulary type {t} vocab {V} top {n_top}", flush=True)
    rng = np.random.default_rng([t, V, n_top])
    few = np.full(V, -np.inf)
    few[rng.permutation(V)[:n_top // 2]] = rng.normal(size=n_top // 2)
    crowd = rng.normal(size=V)
    crowd[V // 2:V // 2 + 2 * n_top] += 20  # next to one another
    nan = rng.normal(size=V)
    nan[rng.permutation(V)[:V // 3]] = np.nan
    rows = np.stack([3 * rng.normal(size=V), np.sort(rng.normal(size=V)), np.sort(rng.normal(size=V))[::-1], np.zeros(V),
                     rng.integers(0, 4, V), few, crowd, nan, np.full(V, -np.inf), np.sort(rng.integers(0, 2, V))])
    raw = S.encode(rows, t)
    tokens = rng.integers(0, V, len(rows))
    S.check_logprobs(S.decode(raw, t), raw, t, tokens, n_top, 1.0)
    pick = rng.integers(0, len(rows), 300)
    a, b = S.run_logprobs(raw, t, V, tokens, n_top, 1.0), S.run_logprobs(raw[pick], t, V, tokens[pick], n_top, 1.0)
    for x, y in zip(a, b):
        np.testing.assert_array_equal(y, x[pick])


def test_largest_of_more_rows_than_a_grid_line(device):
    """Rows past what one dimension of a grid holds in workgroups of sixteen waves."""
    rng = np.random.default_rng(3)
    rows, V, n_top = (1 << 22) + 3, 5, 2
    x = rng.permuted(np.broadcast_to(np.arange(V, dtype=np.float16), (rows, V)), axis=1)
    lp, ent, idx, top = S.run_logprobs(x, F16, V, np.zeros(rows), n_top, 1.0)
    lse = np.log(np.exp(np.arange(V) - (V - 1.0)).sum())
    assert np.array_equal(idx, np.argsort(-x.astype(np.float32), axis=1, kind="stable")[:, :n_top])
    np.testing.assert_allclose(top, np.broadcast_to([-lse, -lse - 1], (rows, 2)), rtol=48 * U)
    np.testing.assert_allclose(lp, x[:, 0].astype(np.float64) - (V - 1) - lse, rtol=48 * U)


@pytest.mark.parametrize("layout", [K.ROPE_HALF, K.ROPE_INTERLEAVED])
def test_rotation_near_the_axes(device, layout):
    """Angles next to multiples of pi/2, where one of cos and sin is all remainder: the
    pair (1, 0) turned by angles that no f32 holds comes out with the f32 functions'
    own error (2 U relative, a step) and the remainder's two roundings (2 U more),
    not with the angle's rounding (up to 2^-23 whatever the result)."""
    D = 128
    rng = np.random.default_rng(layout)
    pos = np.array([1, 3, 1000, 77777, 1 << 20])
    k = rng.integers(1, 9, D // 2)
    for p in pos:
        angle = k * (np.pi / 2) + rng.uniform(-1, 1, D // 2) * 10.0 ** rng.uniform(-6, -0.5, D // 2)
        inv = angle / p  # (f64: p * inv is the angle to 2^-52)
        x = np.zeros((1, 1, D), np.float32)
        if layout == K.ROPE_HALF:
            x[..., :D // 2] = 1
        else:
            x[..., 0::2] = 1
        out = K.DeviceBuffer(x.nbytes)
        K.rope(F32, S.put(x), None, S.i32([p]), S.put(inv), 1, 1, 0, D, q_out=out, layout=layout)
        y = out.download(np.float32).astype(np.float64)
        c, s = (y[:D // 2], y[D // 2:]) if layout == K.ROPE_HALF else (y[0::2], y[1::2])
        th = p * inv
        for got, want, what in ((c, np.cos(th), "cos"), (s, np.sin(th), "sin")):
            S.close(got, want, 4 * U * np.abs(want) + 1e-14, f"{what} at {p}")


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("D,n_rot", [(128, 128), (64, 24)])
@pytest.mark.parametrize("eps", [1e-6, 0.0])
def test_norms_of_any_size(device, t, D, n_rot, eps):
    """Heads whose squares f32 does not hold, beside ordinary ones: normalised all the same."""
    rng = np.random.default_rng([t, D, n_rot])
    sizes = [0, 66, 100, 125, -20, 0, -66, -100, -130]
    rows, nh, nk = len(sizes), 9, 3
    x = np.clip(rng.normal(size=(rows, nh + nk, D)), -3.9, 3.9) * 2.0 ** np.array(sizes)[:, None, None]
    x[:, 1::4] = np.clip(rng.normal(size=x[:, 1::4].shape), -3.9, 3.9)
    raw = S.encode(x.reshape(rows, -1), t)
    x = S.decode(raw, t).reshape(x.shape)
    w = [(1 + 0.1 * rng.normal(size=D)).astype(np.float32) for _ in range(2)]
    inv, ms = K.rope_freqs(n_rot, 1e6)
    pos = rng.integers(0, 40000, rows)
    stride, eps32 = (nh + nk) * D, float(np.float32(eps))
    for norms in ((True, True), (True, False), (False, True)):
        buf = S.put(raw)
        K.rope(t, buf.ptr, buf.ptr + nh * D * raw.itemsize, S.i32(pos), S.put(inv), rows, nh, nk, D, n_rot=n_rot,
               q_norm=S.put(w[0]) if norms[0] else None, k_norm=S.put(w[1]) if norms[1] else None, eps=eps, q_stride=stride, k_stride=stride)
        got = S.decode(buf.download(S.np_type(t), raw.size), t).reshape(x.shape)
        for part, wt, on in ((slice(0, nh), w[0], norms[0]), (slice(nh, None), w[1], norms[1])):
            wt = wt.astype(np.float64) if on else None
            want = S.rope64(x[:, part], wt, pos, inv, ms, n_rot, K.ROPE_HALF, eps32)
            S.close(got[:, part], want, S.rope_bound(want, x[:, part], wt, ms, t, eps32), f"norms {norms}")


@pytest.mark.parametrize("fmt", [K.KV_F8, K.KV_I8])
@pytest.mark.parametrize("nh,T,bound_p", TILES + [(4, 3, 12000)])
@pytest.mark.parametrize("power", [-20, 8, 45, 90])
def test_unit_of_values_leaves_the_result(device, fmt, nh, T, bound_p, power):
    """Values times a power of two: the same codes, and the result times it to the last
    roundings (each of a wave's and a split's two factors 2 U at most, of 16 joined)."""
    rng = np.random.default_rng([fmt, nh, T])
    D, P = 64, 900
    k, v = rng.normal(size=(2, 1, P + T, 1, D))
    q = rng.normal(size=(1, T, nh, D)).astype(np.float32).astype(np.float64)
    sees = S.tree_bits(rng, T)[None]
    out = []
    for z in (0, power):
        c = K.KvCache.allocate(fmt, 1, 1, max(bound_p, P) + T, D)
        kv = S.store_prefix(c, [k, v * 2.0 ** z], P + T)
        out.append(S.run_tree(c, F32, q, T, [P], None, sees, nh, max_prefix=max(bound_p, P))[0] * 2.0 ** -z)
    p = S.tree64(q, [kv[0], np.abs(kv[1]) * 2.0 ** -power], [P], [T], sees, D ** -0.5, F32)[0]  # sum of shares times |values|
    S.close(out[1], out[0], 8 * U * p, "unit")
