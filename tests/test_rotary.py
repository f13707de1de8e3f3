"""Head norms + position rotation against the definition in 64 bits.

Tolerances: fp32 arithmetic on values up to a few units, with an angle exact
to about 2^-24 turns, leaves at most 2e-6 of a head's largest value; the
output's one rounding adds at most the type's unit roundoff, eps / 2, relative."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from oracle import attention as oa


def close(got, want, dtype):
    want = want.double()
    err = (got.double().cpu() - want).abs()
    bound = 1.01 * torch.finfo(dtype).eps / 2 * want.abs() + 4e-6 * want.abs().amax(-1, keepdim=True) + 1e-7
    assert bool((err <= bound).all()), float((err / bound).max())


def make(T, hq, hk, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn((T, hq + 2 * hk, D), generator=g).to(dtype)
    return qkv, 1.0 + 0.3 * torch.randn(D, generator=g), 0.3 * torch.randn(D, generator=g)


def test_scaling_formulas():
    from voom_b200.runtime.rotary import _scaled

    r, theta = 64, 10000.0
    base = [theta ** (-2.0 * i / r) for i in range(r // 2)]
    f, a = _scaled(base, r, theta, {"rope_type": "linear", "factor": 4.0})
    assert a == 1.0 and all(math.isclose(x, y / 4) for x, y in zip(f, base))
    f, a = _scaled(base, r, theta, {"rope_type": "ntk", "factor": 4.0})
    assert f[0] == 1.0 and math.isclose(f[-1], base[-1] / 4, rel_tol=1e-12)  # the slowest pair is stretched in full
    f, a = _scaled(base, r, theta, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 2048})
    assert f[0] == base[0] and math.isclose(f[-1], base[-1] / 4) and math.isclose(a, 0.1 * math.log(4.0) + 1.0)
    assert all(y / 4 <= x <= y for x, y in zip(f, base))
    f, a = _scaled(base, r, theta, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0,
                                    "high_freq_factor": 4.0, "original_max_position_embeddings": 8192})
    for x, y in zip(f, base):
        turns = 8192 * y / (2 * math.pi)
        want = y if turns > 4 else y / 8 if turns < 1 else y / 8 * (4 - turns) / 3 + y * (turns - 1) / 3
        assert math.isclose(x, want, rel_tol=1e-12)
    with pytest.raises(ValueError, match="unknown rotary scaling"):
        _scaled(base, r, theta, {"rope_type": "other", "factor": 2.0})
    with pytest.raises(ValueError, match="at least 1"):
        _scaled(base, r, theta, {"rope_type": "linear", "factor": 0.5})


def test_c_entry_refuses_bad_arguments(built_lib):
    from voom_b200._lib import QkNormRopeArgs

    a = QkNormRopeArgs()
    assert built_lib.voom_qk_norm_rope(None, None) == -1
    assert built_lib.voom_qk_norm_rope(ctypes.byref(a), None) == -1
    for f in ("q", "k", "q_out", "k_out", "pos", "turns"):
        setattr(a, f, 4096)
    a.T, a.hq, a.hk, a.D, a.rot = 1, 1, 1, 64, 63
    assert built_lib.voom_qk_norm_rope(ctypes.byref(a), None) == -1  # an odd rotated part
    a.rot = 66
    assert built_lib.voom_qk_norm_rope(ctypes.byref(a), None) == -1  # more than the head
    a.D, a.rot = 1024, 64
    assert built_lib.voom_qk_norm_rope(ctypes.byref(a), None) == -4  # a head too large
    a.D, a.T = 64, 0
    assert built_lib.voom_qk_norm_rope(ctypes.byref(a), None) == 0   # nothing to do


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,hq,hk,D,rot,layout,norm,zero,wtype", [
    (1, 9, 3, 64, 64, "half", False, False, None),
    (1, 1, 1, 128, 128, "interleaved", True, False, "same"),
    (37, 32, 8, 128, 128, "half", True, False, "same"),
    (300, 4, 1, 256, 64, "interleaved", True, True, "same"),
    (19, 6, 2, 80, 32, "half", True, False, "fp32"),
    (5, 3, 3, 96, 40, "half", True, False, "fp32"),         # chunks of one pair only
    (5, 3, 3, 96, 6, "interleaved", True, False, "fp32"),
    (4, 2, 1, 50, 50, "half", True, True, "fp32"),          # odd half: single values
    (3, 2, 1, 512, 512, "half", True, False, "same"),
    (3, 2, 1, 128, 0, "half", True, False, "same"),         # norms alone
    (2500, 5, 1, 64, 32, "half", True, False, "same"),      # several tokens to a block
])
def test_against_definition(dtype, T, hq, hk, D, rot, layout, norm, zero, wtype):
    from voom_b200.runtime import rotary

    qkv, qw, kw = make(T, hq, hk, D, dtype)
    if zero:
        qw = qw - 1.0
    wt = torch.float32 if wtype == "fp32" else dtype
    qw, kw = qw.to(wt), kw.to(wt)
    pos = torch.randint(0, 5000, (T,), generator=torch.Generator().manual_seed(1))
    plan = rotary.Rotary(D, rot_dim=rot, theta=5e5, layout=layout, device="cuda",
                         scaling={"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 1024}
                         if rot == D and layout == "half" else None)
    d = qkv.cuda()
    q, k = d[:, :hq], d[:, hq:hq + hk]
    kwargs = dict(q_weight=qw.cuda(), k_weight=kw.cuda(), zero_centered=zero) if norm else {}
    gq, gk = rotary.qk_norm_rope(q, k, pos.cuda(), plan, **kwargs)
    for got, x, w in ((gq, qkv[:, :hq], qw), (gk, qkv[:, hq:hq + hk], kw)):
        close(got, oa.norm_rope(x, pos, plan.freqs, rot=rot, layout=layout, factor=plan.factor,
                                weight=w if norm else None, zero_centered=zero), dtype)
    # in place, and into strided outputs, with 32-bit positions: the same bits
    big = torch.full((T, hq + hk + 1, D), 7.0, dtype=dtype, device="cuda")
    rotary.qk_norm_rope(q, k, pos.int().cuda(), plan, out_q=big[:, :hq], out_k=big[:, hq:hq + hk], **kwargs)
    assert torch.equal(big[:, :hq], gq) and torch.equal(big[:, hq:hq + hk], gk) and bool((big[:, -1] == 7.0).all())
    rotary.qk_norm_rope(q, k, pos.cuda(), plan, out_q=q, out_k=k, **kwargs)
    assert torch.equal(d[:, :hq], gq) and torch.equal(d[:, hq:hq + hk], gk)
    assert torch.equal(d[:, hq + hk:].cpu(), qkv[:, hq + hk:])


@pytest.mark.gpu
def test_far_positions_and_odd_alignment():
    from voom_b200.runtime import rotary

    pos = torch.tensor([0, 1, 10 ** 6, 2 ** 31 + 5, -3])
    base = torch.randn(5 * 2 * 64 + 3, generator=torch.Generator().manual_seed(2))
    x = base[3:].view(5, 2, 64)
    plan = rotary.Rotary(64, device="cuda")
    d = base.cuda()[3:].view(5, 2, 64)  # rows on 4 bytes, not on 16
    got, _ = rotary.qk_norm_rope(d, d[:, :1], pos.cuda(), plan)
    close(got, oa.norm_rope(x, pos, plan.freqs, rot=64), torch.float32)


@pytest.mark.gpu
def test_only_one_side_normed_zero_rows_and_empty():
    from voom_b200.runtime import rotary

    qkv, qw, _ = make(6, 2, 1, 64, torch.float32)
    qkv[2] = 0.0
    plan = rotary.Rotary(64, device="cuda")
    d = qkv.cuda()
    pos = torch.arange(6)
    gq, gk = rotary.qk_norm_rope(d[:, :2], d[:, 2:3], pos.cuda(), plan, q_weight=qw.cuda())
    close(gq, oa.norm_rope(qkv[:, :2], pos, plan.freqs, rot=64, weight=qw), torch.float32)
    close(gk, oa.norm_rope(qkv[:, 2:3], pos, plan.freqs, rot=64), torch.float32)
    assert bool((gq[2] == 0).all())
    e, _ = rotary.qk_norm_rope(d[:0, :2], d[:0, 2:3], pos[:0].cuda(), plan)
    assert e.shape == (0, 2, 64)


@pytest.mark.gpu
def test_refusals():
    from voom_b200.runtime import rotary

    with pytest.raises(ValueError, match="even number"):
        rotary.Rotary(64, rot_dim=33, device="cuda")
    with pytest.raises(ValueError, match="head size"):
        rotary.Rotary(1024, device="cuda")
    with pytest.raises(ValueError, match="layout"):
        rotary.Rotary(64, layout="other", device="cuda")
    plan = rotary.Rotary(64, device="cuda")
    q = torch.zeros((2, 2, 64), device="cuda")
    pos = torch.arange(2, device="cuda")
    with pytest.raises(ValueError, match="must both be"):
        rotary.qk_norm_rope(q, q.half(), pos, plan)
    with pytest.raises(ValueError, match="tokens"):
        rotary.qk_norm_rope(q, q, pos[:1], plan)
    with pytest.raises(ValueError, match="int32 or int64"):
        rotary.qk_norm_rope(q, q, pos.float(), plan)
    with pytest.raises(ValueError, match="contiguous"):
        rotary.qk_norm_rope(q.transpose(1, 2).contiguous().transpose(1, 2), q, pos, plan)
    with pytest.raises(ValueError, match="weights"):
        rotary.qk_norm_rope(q, q, pos, plan, q_weight=torch.ones(32, device="cuda"))
    with pytest.raises(ValueError, match="out_q"):
        rotary.qk_norm_rope(q, q, pos, plan, out_q=q[:1])
    with pytest.raises(ValueError, match="device"):
        rotary.qk_norm_rope(q.cpu(), q, pos, plan)
