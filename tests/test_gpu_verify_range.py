"""kq_verify where what is left of a row is of the size of its sum's rounding."""
import numpy as np
import pytest

from test_gpu_verify import call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [3, 5000])
def test_every_likely_id_is_refused(dev, V):
    """Three ids of a row have a probability, each a ten-millionth of the one before, and all are drafted.  Random numbers just below 1
    refuse the first two; what is left is the third's 2^-46 of the row, no more than the 4e-14 to which a weight is known: it is
    taken, or refused too, and then the token is drawn from the row itself.  There always is one."""
    B, T = 256, 4
    rng = np.random.default_rng(0)
    ids = np.array([0, 1, 2]) if V == 3 else np.array([40, 41, 4100])
    x = np.full((B, T, V), -np.inf, np.float32)
    x[:, :, ids] = np.log([1.0, 2.0 ** -23, 2.0 ** -46]) + 0.1 * rng.random((B, 1, 3))
    x[:, :, ids[0]] = 0
    tokens = np.tile(np.concatenate([[0], ids]).astype(np.int32), (B, 1))
    parents = np.array([[-1, 0, 0, 0]], np.int32)
    u = np.full((B, T), 1 - 2.0 ** -24, np.float32)
    u[:, 0] = rng.random(B)
    accepted, path, token = call(dev, x.reshape(-1, V), tokens, parents, u)
    assert set(token) <= set(ids.tolist())
    assert all(a == 0 or p[1] == 3 for a, p in zip(accepted, path))
