"""What the tests of the operators on device tensors share."""
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rounding(t):
    """Largest relative error of one rounding to t, and the absolute one among its subnormal numbers."""
    f = torch.finfo(t)
    return f.eps / 2, f.smallest_normal * f.eps / 2


def assert_near(got, want, slack, what):
    """|got - want| within one rounding to got's type plus `slack` (float64: the arithmetic's own error), element by element; NaN and infinities have to be the same."""
    assert got.shape == want.shape, what
    g, rel_abs = got.double(), rounding(got.dtype)
    rel, small = rel_abs if got.dtype != torch.float32 else (0.0, 0.0)      # (float32: the last rounding is part of the arithmetic)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(want), torch.isnan(g)), what
    assert torch.equal(want[~fine & ~torch.isnan(want)], g[~fine & ~torch.isnan(want)]), what
    slack = torch.as_tensor(slack, dtype=torch.float64, device=want.device).expand_as(want)
    bound = rel * (want.abs() + slack) + slack + small
    over = ((g - want).abs() - bound)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0.0, f"{what}: {float((g - want).abs()[fine].max()):.3g} off, {float(over.max()):.3g} over the bound"
