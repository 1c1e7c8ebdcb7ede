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
