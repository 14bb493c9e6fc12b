"""Type of a result that is asked for twice: by the tensor that is passed and by name."""
import pytest
import torch

import turbofno_amd as tf
from turbofno_amd import api

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("compiled", [True, False])
def test_8bit_result_of_another_type_than_named(compiled, monkeypatch):
    if not compiled:
        monkeypatch.setattr(api, "_operands", None)
    eight = torch.float8_e4m3fn
    xq, Wq = torch.ones(5, 40, device="cuda").to(eight), torch.ones(3, 5, device="cuda").to(eight)
    xs, ws, y = torch.ones(40, device="cuda"), torch.ones(3, device="cuda"), torch.zeros(3, 40, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(TypeError, match="y must be a torch.float32"):
        tf.mix_8bit(xq, xs, Wq, ws, y=y, dtype=torch.float32)
    assert (y == 0).all()
    assert tf.mix_8bit(xq, xs, Wq, ws, y=y, dtype=torch.bfloat16) is y and (y == 5).all()
    assert tf.mix_8bit(xq, xs, Wq, ws, y=y) is y
