"""Scores of more tokens than the workspace has room for at a time, against 64 bits at the ends of the runs and between.  Tolerances: test_gpu_loss."""
import numpy as np
import pytest

from experts_oracle import KINDS, upload
from loss_choice import score_run
from test_gpu_loss import _make
from test_gpu_loss_every_token import _check_all

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,vocabulary,width,kind,vector", [(20000, 128256, 8, "bf16", True), (40001, 128256, 8, "f16", True), (5000, 120007, 7, "f16", False)])
def test_runs_of_tokens(gpu, tokens, vocabulary, width, kind, vector):
    C, kind = gpu.LOSS, KINDS[kind]
    run, _ = score_run(gpu, tokens, vocabulary, width, vector)
    assert tokens / 4 < run < tokens and tokens % run
    x, w, targets, _ = _make(tokens, tokens, vocabulary, width, kind)
    losses, lse = (upload(gpu, np.full(tokens + 5, 7.0, np.float32)) for _ in range(2))
    need = C.cross_entropy_workspace(tokens, vocabulary, width)
    space = gpu.DeviceArray.undef(np.uint8, need + (1 << 20))
    space.fill_bytes(0xFF)

    class Inside:
        _as_parameter_, nbytes = space.ptr, need

    operands = upload(gpu, kind.store(x)), upload(gpu, kind.store(w)), upload(gpu, targets)
    C.cross_entropy(*operands, losses, lse, tokens=tokens, vocabulary=vocabulary, width=width, dtype=kind.marker(gpu), workspace=Inside)
    gpu.synchronize()
    assert np.all(space.to_host()[need:] == 0xFF)
    got = [a.to_host().astype(np.float64) for a in (losses, lse)]
    assert all(np.all(a[tokens:] == 7) and np.all(np.isfinite(a)) for a in got) and not (got[1][:tokens] == 7).any()
    # both sides of where each run begins and of where the last one does, and others
    ends = [e + d for e in (*range(0, tokens, run), tokens - run, tokens) for d in (-2, -1, 0, 1) if 0 <= e + d < tokens]
    some = np.unique(ends + list(np.random.default_rng(1).integers(0, tokens, 150)))
    _check_all([a[some] for a in got], x[some], w, targets[some], None, kind)
    # fewer tokens in the same workspace; tokens' values do not hang on the others
    few = tokens // 3
    C.cross_entropy(*operands, losses, lse, tokens=few, vocabulary=vocabulary, width=width, dtype=kind.marker(gpu), workspace=Inside)
    again = [a.to_host().astype(np.float64) for a in (losses, lse)]
    assert all(np.array_equal(a[few:], b[few:]) for a, b in zip(got, again)) and all(np.all(np.abs(a - b) < 2.0 ** -13) for a, b in zip(got, again))
