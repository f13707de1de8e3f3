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


def _base(r=64, theta=10000.0):
    return [theta ** (-2.0 * i / r) for i in range(r // 2)]


def test_yarn_keys_of_model_configurations():
    from voom_b200.runtime.rotary import _scaled

    r, theta, factor, orig = 64, 10000.0, 40.0, 4096
    yarn = {"rope_type": "yarn", "factor": factor, "original_max_position_embeddings": orig}
    f, a = _scaled(_base(), r, theta, yarn)

    def gain(m):
        return 0.1 * m * math.log(factor) + 1.0

    assert math.isclose(a, gain(1.0))
    assert math.isclose(_scaled(_base(), r, theta, {**yarn, "mscale": 1.0, "mscale_all_dim": 1.0})[1], 1.0)
    assert math.isclose(_scaled(_base(), r, theta, {**yarn, "mscale": 0.707, "mscale_all_dim": 0.5})[1], gain(0.707) / gain(0.5))
    assert _scaled(_base(), r, theta, {**yarn, "mscale": 0.707, "mscale_all_dim": 0.5, "attention_factor": 1.5})[1] == 1.5
    with pytest.raises(ValueError, match="together"):
        _scaled(_base(), r, theta, {**yarn, "mscale": 0.707})
    # the ramp between the pairs that make 32 turns and 1 turn over the original context, not rounded to whole pairs
    g, _ = _scaled(_base(), r, theta, {**yarn, "truncate": False})
    ends = [r * math.log(orig / (t * 2 * math.pi)) / (2 * math.log(theta)) for t in (32.0, 1.0)]
    for i, (x, y) in enumerate(zip(g, _base())):
        ramp = min(max((i - ends[0]) / (ends[1] - ends[0]), 0.0), 1.0)
        assert math.isclose(x, y / factor * ramp + y * (1.0 - ramp), rel_tol=1e-12)
    assert g != f and _scaled(_base(), r, theta, {**yarn, "truncate": True})[0] == f


def test_default_scaling_and_keys_that_would_be_ignored():
    from voom_b200.runtime.rotary import _scaled

    assert _scaled(_base(), 64, 10000.0, {"rope_type": "default"}) == (_base(), 1.0)
    assert _scaled(_base(), 64, 10000.0, {"rope_type": "default", "rope_theta": 10000.0}) == (_base(), 1.0)
    assert _scaled(_base(), 64, 10000.0, {"type": "linear", "factor": 2, "truncate": None})[1] == 1.0
    for scaling in ({"rope_type": "default", "factor": 2.0}, {"rope_type": "default", "rope_theta": 5e5},
                    {"rope_type": "linear", "factor": 2.0, "mscale": 1.0},
                    {"rope_type": "llama3", "factor": 2.0, "beta_fast": 32},
                    {"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 4096, "other": 1}):
        with pytest.raises(ValueError, match="rotary scaling"):
            _scaled(_base(), 64, 10000.0, scaling)
    half = {"rope_type": "default", "partial_rotary_factor": 0.5}
    assert _scaled(_base(), 64, 10000.0, half, 128) == (_base(), 1.0)
    with pytest.raises(ValueError, match="rotary scaling"):
        _scaled(_base(), 64, 10000.0, half, 64)


def test_c_entry_takes_one_side_alone(built_lib):
    import ctypes

    from voom_b200._lib import QkNormRopeArgs

    a = QkNormRopeArgs()
    for f in ("q", "q_out", "pos", "turns"):
        setattr(a, f, 4096)
    a.T, a.hq, a.hk, a.D, a.rot = 0, 1, 0, 64, 64
    assert built_lib.voom_qk_norm_rope(ctypes.byref(a), None) == 0  # no key heads: no keys
    a.hk = 1
    assert built_lib.voom_qk_norm_rope(ctypes.byref(a), None) == -1
    a.hq, a.k, a.k_out, a.q, a.q_out = 0, 4096, 4096, None, None
    assert built_lib.voom_qk_norm_rope(ctypes.byref(a), None) == 0  # no query heads: no queries


@pytest.mark.gpu
def test_queries_or_keys_alone():
    from voom_b200.runtime import rotary

    x = torch.randn((4, 3, 64), generator=torch.Generator().manual_seed(3))
    pos = torch.arange(4)
    plan = rotary.Rotary(64, device="cuda")
    d = x.cuda()
    want = oa.norm_rope(x, pos, plan.freqs, rot=64)
    q, k = rotary.qk_norm_rope(d, d[:, :0], pos.cuda(), plan)
    close(q, want, torch.float32)
    assert k.shape == (4, 0, 64)
    q, k = rotary.qk_norm_rope(d[:, :0], d, pos.cuda(), plan)
    close(k, want, torch.float32)
    assert q.shape == (4, 0, 64)
