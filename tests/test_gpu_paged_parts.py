"""Parts of a long cache in which a row has no score but -inf: what its values of v make of it
does not go by how many parts the keys are cut into."""
import numpy as np
import pytest

import attention_ref as A
import operators_ref as R
from test_gpu_paged_attention import Cache

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("lens,bad", [(200, 60), (2000, 600), (2000, 1900)])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_a_value_that_is_not_finite_stays_in_the_sum(value, lens, bad, new, dt):
    """0 times it: one v among the `bad` positions whose scores are -inf, one part or eight."""
    c = Cache([lens], [new], 2, 1, 16, 16, dt)
    c.q = R.rounded(np.abs(c.q) + 1, dt)
    c.k[0][:bad] = -np.inf
    c.v[0][5, 0, 3] = value
    o = c.attend(0.1)
    assert np.isnan(o[:, :, 3]).all()
    first = lens - bad - new
    for h in range(2):
        k, v = (t[0][bad:, 0].astype(np.float64) for t in (c.k, c.v))
        want, bound, *_ = A.attend(c.q[:, h].astype(np.float64), k, v, first, 0.1, True, dt)
        rest = np.arange(16) != 3
        R.check(o[:, h][:, rest], want[:, rest], bound[:, rest], f"head {h}")
