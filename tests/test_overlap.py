"""Outputs that overlap themselves, or what is still read, are refused.

The checks (voom_b200/csrc/rows.h, compiled for the host) against sets of
elements: they may refuse an odd interleaving, never accept an overlap, and have
to accept what projections and caches look like."""

from __future__ import annotations

import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

HERE = Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def rows(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    out = tmp_path_factory.mktemp("rows") / "librows_host.so"
    subprocess.run([cxx, "-O2", "-std=c++17", "-shared", "-fPIC", str(HERE / "native" / "rows_host.cpp"), "-o", str(out)],
                   check=True)
    return ctypes.CDLL(str(out))


def _arg(t):
    return (ctypes.c_int64 * 8)(*t)


def _elements(t):
    at, n0, n1, n2, s0, s1, s2, run = t
    return [at // 2 + i * s0 + j * s1 + k * s2 + e
            for i in range(n0) for j in range(n1) for k in range(n2) for e in range(run)]


def test_no_overlap_is_accepted(rows):
    r = random.Random(1)
    told = [0, 0, 0, 0]
    for _ in range(20000):
        a, b = ((2 * r.randrange(500, 560), r.randrange(0, 4), r.randrange(1, 4), r.randrange(1, 4), r.choice((0, 6, 24, 48, 60)),
                 r.choice((-12, 2, 8, 12, 24)), r.choice((-4, 0, 2, 4, 5)), r.randrange(1, 5)) for _ in range(2))
        x, y = _elements(a), _elements(b)
        separate, disjoint = rows.rows_separate(_arg(a)), rows.rows_disjoint(_arg(a), _arg(b))
        assert not separate or len(set(x)) == len(x), a
        assert not disjoint or not set(x) & set(y), (a, b)
        told[separate] += 1
        told[2 + disjoint] += 1
    assert min(told) > 500


def test_layouts_of_projections_and_caches_are_accepted(rows):
    hq, hk, D, B, n = 8, 2, 64, 3, 5
    W = (hq + 2 * hk) * D  # a token of the fused projection
    fused = [(4096 + 2 * at * D, B, n, h, n * W, W, D, D) for at, h in ((0, hq), (hq, hk), (hq + hk, hk))]
    heads_first = [(4096 + 2 * at * n * D, B, n, h, n * W, D, n * D, D) for at, h in ((0, hq), (hq, hk), (hq + hk, hk))]
    for parts in (fused, heads_first):
        for i, a in enumerate(parts):
            assert rows.rows_separate(_arg(a))
            for j, b in enumerate(parts):
                assert bool(rows.rows_disjoint(_arg(a), _arg(b))) == (i != j)
    whole = (4096, B, n, hq + 2 * hk, n * W, W, D, D)
    assert not rows.rows_disjoint(_arg(whole), _arg(fused[1]))
    assert rows.rows_separate(_arg((4096, 1, 1, hq, 0, 0, D, D)))  # strides of single items do not count
    assert not rows.rows_separate(_arg((4096, B, n, hq, 0, W, D, D))) and not rows.rows_separate(_arg((4096, B, n, hq, n * W, W, D - 8, D)))
    far = 1 << 62  # products of strides and counts pass 64 bits
    assert rows.rows_separate(_arg((4096, 4, 4, 4, far, far // 8, 64, 64)))


def test_c_entries_refuse_overlaps(built_lib):
    from voom_b200._lib import KvViewStruct, QkNormRopeArgs, TreeAttentionArgs

    c = KvViewStruct()
    c.k = c.v = c.len = 1 << 30
    c.k_page = c.k_head = c.v_page = c.v_head = 64 * 64
    c.k_pos = c.v_pos = 64
    c.B, c.hk, c.D, c.page, c.max_len = 2, 2, 64, 64, 64

    def attn(**kw):
        """-5 where it is refused; else whether the call goes on to its scratch."""
        a = TreeAttentionArgs()
        a.q, a.kn, a.vn, a.out, a.weights = 1 << 20, 1 << 21, 1 << 22, 1 << 23, 1 << 24
        a.n, a.hq, a.scale = 3, 4, 0.125
        a.q_h = a.kn_h = a.vn_h = a.o_h = 64
        a.q_t = a.o_t = 4 * 64
        a.kn_t = a.vn_t = 2 * 64
        a.q_b = a.o_b = 3 * 4 * 64
        a.kn_b = a.vn_b = 3 * 2 * 64
        a.w_b, a.w_h = 2 * 80, 80
        for x, y in kw.items():
            setattr(a, x, y)
        if built_lib.voom_tree_attention_scratch_bytes(ctypes.byref(c), ctypes.byref(a)):
            return 1
        return built_lib.voom_tree_attention(ctypes.byref(c), ctypes.byref(a), None, 0, None)

    assert attn() == 1 and attn(weights=None, w_b=0, w_h=0, lse=None) != -5
    assert attn(out=1 << 20) == -5 and attn(out=(1 << 20) + 128) == -5  # q, or part of it
    assert attn(out=1 << 21) == -5 and attn(out=(1 << 22) - 256) == -5
    assert attn(o_b=0) == -5 and attn(o_t=0) == -5 and attn(o_h=0) == -5 and attn(o_t=128) == -5
    assert attn(w_b=0) == -5 and attn(w_h=0) == -5 and attn(w_h=66) == -5
    assert attn(w_h=67, w_b=134) == 1  # rows of max_len + n weights, one after another

    a = QkNormRopeArgs()
    a.pos = a.turns = 4096
    a.T, a.hq, a.hk, a.D, a.rot = 3, 4, 2, 64, 64
    for name, at, heads in (("q", 20, 4), ("k", 21, 2), ("qo", 22, 4), ("ko", 23, 2)):
        setattr(a, {"qo": "q_out", "ko": "k_out"}.get(name, name), 1 << at)
        setattr(a, name + "_token", heads * 64)
        setattr(a, name + "_head", 64)

    def rope(**kw):
        b = QkNormRopeArgs.from_buffer_copy(a)
        for x, y in kw.items():
            setattr(b, x, y)
        return built_lib.voom_qk_norm_rope(ctypes.byref(b), None)

    assert rope(qo_token=0) == -5 and rope(ko_head=0) == -5 and rope(qo_head=32) == -5
    assert rope(q_out=(1 << 20) + 128) == -5 and rope(q_out=1 << 21) == -5 and rope(k_out=1 << 20) == -5
    assert rope(q_out=1 << 20, qo_token=8 * 64) == -5  # q's place in other strides
    assert rope(k_out=1 << 22) == -5  # both outputs


@pytest.mark.gpu
def test_overlaps_are_refused_and_fused_layouts_are_not():
    from voom_b200.runtime import kv_attention as kva
    from voom_b200.runtime import rotary

    x = torch.randn((1, 5, 8, 64), device="cuda").to(torch.bfloat16)
    k = torch.randn((1, 2, 30, 64), device="cuda").to(torch.bfloat16)
    view = kva.KVView.contiguous(k, k, torch.tensor([30], dtype=torch.int32, device="cuda"))
    tree = kva.DraftTree.chain(1, 5, "cuda")
    args = (x[:, :, :4], x[:, :, 4:6], x[:, :, 6:], tree, view)
    for out in (x[:, :, :4], x[:, :, 3:7], torch.empty((1, 5, 1, 64), dtype=x.dtype, device="cuda").expand(1, 5, 4, 64)):
        with pytest.raises(ValueError, match="share"):
            kva.tree_attention(*args, out=out)
    with pytest.raises(ValueError, match="share"):
        kva.tree_attention(*args, weights=torch.zeros((1, 1, 40), device="cuda").expand(1, 2, 40))
    wide = torch.zeros((1, 5, 12, 64), dtype=x.dtype, device="cuda")
    wide[:, :, 4:] = x
    got = kva.tree_attention(wide[:, :, 4:8], wide[:, :, 8:10], wide[:, :, 10:], tree, view, out=wide[:, :, :4])
    assert torch.equal(got, kva.tree_attention(*args)) and torch.equal(wide[:, :, 4:], x)
    plan = rotary.Rotary(64, device="cuda")
    pos = torch.arange(5, device="cuda")
    q, kk = x[0, :, :4], x[0, :, 4:6]
    for kw in (dict(out_q=x[0, :, 1:5]), dict(out_k=x[0, :, 0:2]), dict(out_q=x[0, :1, :4].expand(5, 4, 64)),
               dict(out_q=wide[0, :, :4], out_k=wide[0, :, 3:5])):
        with pytest.raises(ValueError, match="overlap"):
            rotary.qk_norm_rope(q, kk, pos, plan, **kw)
    want = rotary.qk_norm_rope(q, kk, pos, plan)
    rotary.qk_norm_rope(q, kk, pos, plan, out_q=q, out_k=kk)
    assert torch.equal(q, want[0]) and torch.equal(kk, want[1])
