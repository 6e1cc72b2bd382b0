"""What the native forms of the operators refuse before a launch, and how the launchers choose, without a GPU."""
import pytest
import torch

BF = torch.bfloat16


def test_operands_on_another_device_are_refused():
    """An address of another device must not reach a kernel."""
    from fbamtrain_b200.ops.feedforward import gated_mlp
    from fbamtrain_b200.ops.native_ops import _need_elem, linear
    here = {"x": torch.zeros(4, 8, dtype=BF), "w_in": torch.zeros(32, 8, dtype=BF), "w_out": torch.zeros(8, 16, dtype=BF),
            "b_in": torch.zeros(32, dtype=BF), "b_out": torch.zeros(8, dtype=BF), "act": "gelu", "residual": torch.zeros(4, 8, dtype=BF)}
    for name in ("x", "w_in", "w_out", "b_in", "b_out", "residual"):
        with pytest.raises(ValueError, match="one device"):
            gated_mlp(**{**here, name: here[name].to("meta")})
    with pytest.raises(ValueError, match="one device"):
        linear(here["x"], here["w_in"].to("meta"))
    with pytest.raises(TypeError, match="one 16-bit type"):
        _need_elem(here["x"], here["w_in"].half())
    assert _need_elem(here["x"], None, here["w_in"]) == BF
