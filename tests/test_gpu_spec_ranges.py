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
TILES = [(4, 3, 300), (8, 4, 300), (16, 4, 320000), (16, 8, 320000)]


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
