"""Head norms + rotation: values that are not finite, and scaling as model
configurations write it."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import attention as oa
from tests.test_rotary import close


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("offset", [0, 2, 1])  # rows on 16 bytes; on one pair; on one value
@pytest.mark.parametrize("D,rot", [(128, 32), (96, 48), (64, 0)])
def test_values_past_the_rotated_part_keep_to_themselves(dtype, layout, offset, D, rot):
    """Without a norm, an infinity or NaN past `rot` changes no other value."""
    from voom_b200.runtime import rotary

    T, H = 3, 5
    base = torch.randn(offset + T * H * D, generator=torch.Generator().manual_seed(1)).to(dtype)
    x = base[offset:].view(T, H, D)
    for h, bad in enumerate((math.inf, -math.inf, math.nan, math.inf)):  # the last head has none
        x[:, h, rot + 1 + 7 * h] = bad
        x[1, h, D - 1 - h] = bad
    d = base.cuda()[offset:].view(T, H, D)
    pos = torch.tensor([0, 5, 1000])
    plan = rotary.Rotary(D, rot_dim=rot, layout=layout, device="cuda")
    got, _ = rotary.qk_norm_rope(d, d[:, :1], pos.cuda(), plan)
    assert torch.equal(got[..., rot:].cpu().nan_to_num(nan=-5.0), x[..., rot:].nan_to_num(nan=-5.0))  # copied
    if rot:
        close(got[..., :rot], oa.norm_rope(x[..., :rot], pos, plan.freqs, rot=rot, layout=layout), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("offset", [0, 2, 1])
def test_an_infinity_in_a_normed_head(layout, offset):
    """x / rms: the infinite value becomes NaN, the unrotated others 0."""
    from voom_b200.runtime import rotary

    D, rot = 128, 32
    base = torch.randn(offset + 2 * D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    d = base.cuda()[offset:].view(1, 2, D)
    d[0, 0, 70] = math.inf
    plan = rotary.Rotary(D, rot_dim=rot, layout=layout, device="cuda")
    got, _ = rotary.qk_norm_rope(d, d[:, :1], torch.tensor([3], device="cuda"), plan, q_weight=torch.ones(D, device="cuda"))
    other = torch.ones(D, dtype=torch.bool)
    other[70] = False
    assert bool(got[0, 0, 70].isnan()) and bool((got[0, 0].cpu()[other] == 0).all())
    assert bool(torch.isfinite(got[0, 1]).all())
