"""Edges of the model-level tuning calls. Tolerances as in tests/test_tuning_step_gpu.py."""
import numpy as np
import pytest

from tests.test_tuning_step_gpu import SPEC, mt, tokens  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("chunk", [0, 7])
@pytest.mark.parametrize("weighted", [False, True])
def test_rows_outside_every_sequence_do_not_count(mt, chunk, weighted):  # noqa: F811
    """Prompt rows before the first answer and padding behind the last, whatever their targets."""
    m = mt.Model(**SPEC, ckpt=1)
    m.set_loss_chunk(chunk)
    ids, targets = tokens(48)
    w = (np.random.RandomState(2).rand(48) > 0.3).astype(np.float32) if weighted else np.ones(48, np.float32)
    w[:5] = w[41:] = 0
    masked = targets.copy()
    masked[:5] = masked[41:] = -100
    seq = [5, 16, 29, 32, 41]
    refp = np.full(48, -5.0)
    want = m.preference_step(ids, targets, seq, 16, ref_logp=refp, weight=w)
    grads = m.grads()
    w[:5] = w[41:] = 1
    got = m.preference_step(ids, masked, seq, 16, ref_logp=refp, weight=w if weighted else None)
    assert got["loss"] == want["loss"] and np.array_equal(got["margin"], want["margin"])
    again = m.grads()
    for n in grads:
        assert np.array_equal(grads[n], again[n]), n
    masked[20] = -100
    w[20] = 1
    with pytest.raises(mt.MtError, match="target out of range"):
        m.preference_step(ids, masked, seq, 16, ref_logp=refp, weight=w if weighted else None)
