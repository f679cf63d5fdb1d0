"""ops.sample's settings, looked at before anything is uploaded (no GPU)."""
import numpy as np
import pytest

from test_sampling_host import built  # noqa: F401  (the fixture)


def test_top_k_that_is_no_whole_number(built, monkeypatch):  # noqa: F811
    """What a conversion to 32 bits would change is refused: a fraction, a number beyond them, one that is none."""
    backend, _, _ = built
    from llamd_rs_b200 import ops

    class Uploaded(Exception):
        pass

    def upload(a):
        raise Uploaded

    monkeypatch.setattr(ops.DevBuf, "from_array", upload)
    x, u = np.zeros((2, 10), np.float32), [0.1, 0.2]
    for k in (2.7, [20, 2.5], 2 ** 32 + 5, [1, 2 ** 31], -2 ** 31 - 1, np.nan, np.inf, "20", np.array([1, 2 ** 40])):
        with pytest.raises(backend.Malformed):
            ops.sample(x, u, top_k=k)
    for k in (None, 20, 20.0, [1, 50], np.int64(7), np.array([0, -3]), 2 ** 31 - 1):
        with pytest.raises(Uploaded):
            ops.sample(x, u, top_k=k)
