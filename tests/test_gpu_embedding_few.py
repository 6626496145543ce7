"""The embedding's gradient on either side of the bounds between its one-launch form
and sorting: positions, bytes of dy, bytes of dw."""
import numpy as np
import pytest

import operators_ref as R
from oxidizedmlx_amd import abi, synth
from test_gpu_embedding import gradient, words

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("kind", ["one id", "words", "each once"])
@pytest.mark.parametrize("n,kib,vocab", [(1, 512, 60), (2, 256, 90), (16, 32, 90), (33, 16, 90), (64, 8, 90), (64, 1, 90),
                                         (65, 1, 90), (1, 256, 150), (16, 16, 2100), (64, 4, 8200)])
@pytest.mark.parametrize("more", [0, 1, 5])
def test_either_side_of_the_bytes_of_dy(n, kib, vocab, more, kind, dt):
    """Rows of `kib` KiB and `more` values: n of them are 512 KiB or just over, or 256
    where dw has more than 32 MiB."""
    dim = kib * 1024 // (4 if dt == abi.F32 else 2) + more
    ids = {"one id": np.full(n, 17), "words": words(n, n, vocab), "each once": (np.arange(n) * 29) % vocab}[kind]
    ids = ids.astype(np.int32)
    dy = R.rounded(synth.normal(n + dim, (n, dim)), dt)
    R.check(gradient(dy, ids, vocab, 0.5, dt), *R.embedding_vjp(dy, ids, vocab, 0.5, dt), f"{n} of {dim} {kind}")


@pytest.mark.parametrize("n", [1, 5, 64])
@pytest.mark.parametrize("vocab", [98304, 98305])
def test_either_side_of_the_bytes_of_dw(n, vocab):
    """98304 rows of 512 f32 values are 192 MiB."""
    ids = np.concatenate([words(n, n, vocab)[:-1], [vocab - 1]]).astype(np.int32)
    dy = synth.normal(n, (n, 512))
    got = gradient(dy, ids, vocab, 2.0, abi.F32)
    some = np.unique(ids)
    want, bound = R.embedding_vjp(dy, np.searchsorted(some, ids), len(some), 2.0, abi.F32)
    R.check(got[some], want, bound, f"{n} ids of {vocab}")
    got[some] = 0.0
    assert not got.any()
