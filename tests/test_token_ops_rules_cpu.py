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


@pytest.mark.parametrize("two_cta,pairs", [("auto", -1), (False, 0), (True, 1)])
def test_the_gated_block_obeys_the_choice_of_pairs(two_cta, pairs, monkeypatch):
    """The fused products take native_ops.TWO_CTA as an argument; where it is not left to the sizes, the plain ones are made by
    `gemm`, which looks at it itself, and the block's entry points get no place to put theirs."""
    from fbamtrain_b200.ops import feedforward, native, native_ops
    calls, products = [], []

    class Library:
        def __getattr__(self, entry):
            return lambda *args: calls.append((entry, args)) or 0

    def product(a, b, **kw):
        products.append(kw)
        return torch.zeros(a.shape[1] if kw.get("a_mn") else a.shape[0], b.shape[1] if kw.get("b_mn") else b.shape[0], dtype=a.dtype)

    monkeypatch.setattr(native, "lib", lambda like=None: Library())
    monkeypatch.setattr(native, "stream", lambda: 0)
    monkeypatch.setattr(native, "status_word", lambda device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(native_ops, "TWO_CTA", two_cta)
    for module in (native_ops, feedforward):
        monkeypatch.setattr(module, "gemm", product)
    x, w_in, w_out = (torch.zeros(*s, dtype=BF).requires_grad_() for s in ((40, 8), (32, 8), (24, 16)))
    y = feedforward.gated_mlp(x, w_in, w_out, None, None, "gelu", None)
    torch.autograd.grad((y,), (x, w_in, w_out), (torch.zeros_like(y),))
    assert [entry for entry, _ in calls] == ["fbam_gated_block_fwd", "fbam_gated_block_bwd"]
    assert [args[-3] for _, args in calls] == [pairs, pairs]
    plain = two_cta == "auto"
    assert len(products) == (0 if plain else 4)
    assert (calls[0][1][12] != 0) == plain and [bool(v) for v in calls[1][1][14:17]] == 3 * [plain]
