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
