"""Distillation with up to 1024 entries of the teacher's at lengths where those decide how a row is cut, against float64."""
import pytest

from tests.test_gpu_op_distill import _case, _check, dev  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("kb,top", [(100, 256), (104, 64), (103, 8), (66, 1024), (70, 1024), (350, 1024), (420, 500)])
def test_against_float64(dev, type, kb, top):  # noqa: F811
    vocab = kb * 1024 // (4 if type == "f32" else 2) - 3
    logits, ids, t, _ = _case(160, vocab, top, type, vocab + top)
    _check(dev, logits, ids, t, 2.0)
