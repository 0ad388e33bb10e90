"""The tensor calls on 8-bit rows and score rows: what they read and refuse, on the host (CPU-safe)."""
import pytest

torch = pytest.importorskip("torch")

from vectordb_amd import scores as S  # noqa: E402


def host_rows(n, dim=32):
    """A Q8Rows of host tensors, made past its own check."""
    r = S.Q8Rows.__new__(S.Q8Rows)
    r.codes, r.scales, r.norms2, r.dim = torch.zeros(n, 32, dtype=torch.uint8), torch.zeros(n, 4, dtype=torch.uint8), torch.zeros(n), dim
    return r


def test_rows_keep_no_address(vdb):
    """What a call hands over is what the tensors are when it is made: nothing of them is kept from an earlier moment."""
    r = host_rows(4)
    assert set(S.Q8Rows.__slots__) == {"codes", "scales", "norms2", "dim"}
    for call in (lambda: S.score_rows(r, r, 1), lambda: r._c):
        with pytest.raises(vdb.ArgumentError, match="codes"):                       # not an AttributeError: the tensors were looked at
            call()
