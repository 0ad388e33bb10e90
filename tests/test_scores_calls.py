"""The tensor calls on 8-bit rows and score rows: what they read and refuse, on the host (CPU-safe)."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from vectordb_amd import scores as S  # noqa: E402
from vectordb_amd.capi import ScoreAdjustC  # noqa: E402


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


@pytest.mark.parametrize("call", [lambda: S.score_rows(1, 2), lambda: S.score_rows(1, 2, 3, 4, 5), lambda: S.score_rows(1, 2, 3, colour=4), lambda: S.score_rows(1, 2, 3, base=4),
                                  lambda: S.quantize_rows(), lambda: S.quantize_rows(rows=1, rown=2), lambda: S.adjust_scores(1), lambda: S.adjust_scores(1, 2, 3), lambda: S.adjust_scores(1, 2, bost=3)])
def test_calls_of_another_form_are_type_errors(call):
    with pytest.raises(TypeError):
        call()


@pytest.mark.parametrize("call", [lambda r: S.quantize_rows(None), lambda r: S.quantize_rows(rows=torch.zeros(2, 4, device="meta")), lambda r: S.score_rows(r, 3, 1), lambda r: S.score_rows(base=r, queries=r, metric=1),
                                  lambda r: S.adjust_scores([[1.0]], 1), lambda r: S.adjust_scores(metric=1, scores=torch.zeros(2, 2)), lambda r: S.Q8Rows.empty(3, 0, "cpu"), lambda r: S.Q8Rows.empty(-1, 8, "cpu"),
                                  lambda r: S.Q8Rows.empty(3, 8, "cpu"), lambda r: S.Q8Rows(1, 2, 3, 4)])
def test_what_is_no_tensor_on_the_gpu_is_refused(vdb, call):
    with pytest.raises(vdb.ArgumentError):
        call(host_rows(4))


def test_the_calls_say_what_they_take():
    import inspect
    assert list(inspect.signature(S.quantize_rows).parameters) == ["rows", "out"]
    assert list(inspect.signature(S.score_rows).parameters) == ["queries", "base", "metric", "out"]
    p = inspect.signature(S.adjust_scores).parameters
    assert list(p) == ["scores", "metric", "pass_bits", "boost", "seen", "seen_offsets", "repeat", "frequency", "presence", "out"]
    assert all(p[k].kind is inspect.Parameter.KEYWORD_ONLY and p[k].default is None for k in list(p)[2:])
    assert all(f.__doc__ for f in (S.quantize_rows, S.score_rows, S.adjust_scores))


@pytest.mark.parametrize("n_seen", [1 << 60, 1 << 62, (1 << 62) + 1, (1 << 64) - 1])
def test_a_list_beyond_the_address_space_is_refused(vdb, n_seen):
    """4 n_seen bytes that wrap to a few must not pass for a short list."""
    p = 1 << 20
    how = ScoreAdjustC(n_seen=n_seen, seen=p + (1 << 31), seen_offsets=p + (1 << 32))
    with pytest.raises(vdb.ArgumentError):
        vdb.check(vdb.fn.score_adjust_dev(p, 100, 4, 100, 1, C.byref(how), p + (1 << 30), 100, None))


def test_the_module_alone_raises_and_does_not_crash():
    """Its functions before vectordb_amd.scores has given it the entry points."""
    import os
    import subprocess
    import sys
    calls = ["quantize_rows(1)", "score_rows(1, 2, 3)", "adjust_scores(1, 2)", "check_rows(1, 2, 3, 4)", "rows_struct(1, 2, 3, 4)", "check_rows(1)", "bind()"]
    code = "import torch\nfrom vectordb_amd import _tensors as t\n" + "".join("try:\n    t.%s\nexcept (RuntimeError, TypeError):\n    print('raised', flush=True)\n" % c for c in calls)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split() == ["raised"] * len(calls), (r.returncode, r.stdout, r.stderr[-500:])
