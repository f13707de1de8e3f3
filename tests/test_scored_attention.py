"""Tree attention with capped, biased and windowed scores, against the definition
in 64 bits.

Tolerances: those of test_kv_attention.py (scores off by 1e-5, lse by 3e-5, a row's
weights by 5e-5, the output by two half units of the type and of max |v|), and what
the cap adds.  cap tanh(z / cap) is computed as cap (1 - 2 r), r = 1 / (1 + u), u =
2^t.  In units of 2^-24: u is off by 4 relative (ex2) and by ln 2 |t| (the rounding
of t), of which r takes u / (1 + u)^2: 1 and 0.23 at most; the rounding of 1 + u
gives r another 1, the reciprocal 2.  So cap 2 dr <= 8.5 cap 2^-24, and the
rounding of the result in log2 units 1.5: 10 cap 2^-24 = 6e-7 cap.  That form is for
|z| > 3/4 cap, where it is at most 8e-7 |z|; below, a polynomial is off by 7.8e-7 of z and
the rounding of x P + bias, 9e-7 |z| in all.  So a capped score is off by 9e-7 min(cap, 20),
as the scores here are below 20 (times `sharp`).  A bias is
rounded to 2^-24 of itself, and of what it is added to: with biases b <= 16 scores
apart from the row's largest counting (e^-16 of the weight past that), 3e-6."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import attention as oa
from oracle import decoding as od
from tests.test_kv_attention import STEP, check, inputs, parents_of, place


def slopes_of(hq):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], dtype=torch.float32)


def run_case(B, n, hq, hk, D, lens, dtype, *, cap=0.0, bias=False, window=0, layout="whole", page=16, kind="tree",
             weights=True, tw=False, seed=0, sharp=1.0):
    from voom_b200.runtime import kv_attention as kva

    qkv, k, v = inputs(B, n, hq, hk, D, lens, dtype, seed)
    qkv[:, :, :hq] *= sharp
    par = [parents_of(kind, n, seed + b) for b in range(B)]
    d = qkv.cuda()
    # what no row sees of a cache, none may feel
    seen = [max(0, x + 1 - window) if window else 0 for x in lens]
    k2, v2 = k.clone(), v.clone()
    for b, s in enumerate(seen):
        k2[b, :, :s] = math.nan
        v2[b, :, :s] = math.inf
    view = place(k2, v2, lens, layout, page)
    tree = kva.DraftTree.chain(B, n, "cuda") if kind == "chain" else kva.DraftTree(
        torch.tensor(par, dtype=torch.int32, device="cuda").reshape(B, n))
    slopes = slopes_of(hq) if bias else None
    w0 = torch.rand((B, hk, view.max_len + n + 3), generator=torch.Generator().manual_seed(9))
    w = w0.cuda() if weights else None
    t = torch.rand((B, n), generator=torch.Generator().manual_seed(8)) if tw else None
    for b in range(B):
        for j in range(n):
            if par[b][j] == -2:
                d[b, j] = math.nan
    args = (d[:, :, :hq], d[:, :, hq:hq + hk], d[:, :, hq + hk:], tree, view)
    kw = dict(cap=cap or None, slopes=None if slopes is None else slopes.cuda(), window=window or None, return_lse=True)
    out, lse = kva.tree_attention(*args, weights=w, token_weight=None if t is None else t.cuda(), **kw)
    bare, bare_lse = kva.tree_attention(*args, **kw)
    torch.cuda.synchronize()
    view.check_status()
    score = 3e-5 * max(1.0, sharp) + 9e-7 * min(cap, 20.0 * max(1.0, sharp)) + (3e-6 if bias else 0.0)
    for b, x in enumerate(lens):
        o, l, s = od.scored_attention(qkv[b, :, :hq], qkv[b, :, hq:hq + hk], qkv[b, :, hq + hk:], oa.tree_sees(par[b]),
                                      oa.tree_depth(par[b]), k[b, :, :x], v[b, :, :x], D ** -0.5, cap=cap, slopes=slopes,
                                      window=window, token_weight=None if t is None else t[b])
        big = max(float(v[b].abs().max()), float(qkv[b, :, hq + hk:].abs().max()))
        tol = (2 * STEP[dtype] + 2 * score) * big
        check(out[b], o, tol, ("out", b))
        check(lse[b], l, score, ("lse", b))
        check(bare[b], o, tol, ("out without weights", b))
        check(bare_lse[b], l, score, ("lse without weights", b))
        if weights:
            want = w0[b].double()
            want[:, :x + n] += s
            check(w[b], want, (2e-5 + score) * max(1.0, sharp) * (n * hq // hk) ** 0.5 + 1e-6, ("weights", b))
    return out, lse, w


KINDS = [dict(cap=5.0), dict(bias=True), dict(window=40), dict(cap=30.0, bias=True, window=70)]


@pytest.mark.gpu
@pytest.mark.parametrize("kw", KINDS)
@pytest.mark.parametrize("dtype,layout,page", [(torch.bfloat16, "whole", 0), (torch.float16, "pool", 16),
                                               (torch.bfloat16, "pool", 5), (torch.float16, "pages", 48)])
@pytest.mark.parametrize("n,hq,hk,D", [(1, 9, 3, 64), (1, 8, 1, 128), (7, 4, 2, 128), (5, 6, 2, 256), (20, 3, 1, 64),
                                       (33, 4, 2, 64), (20, 8, 1, 128), (48, 8, 2, 256)])
def test_kinds_layouts_heads_and_types(kw, dtype, layout, page, n, hq, hk, D):
    run_case(3, n, hq, hk, D, [77, 0, 130], dtype, layout=layout, page=page, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 64, 65, 127, 128, 129, 200, 700, 10 ** 9])
@pytest.mark.parametrize("n,hq,D", [(1, 4, 64), (1, 2, 256), (9, 4, 128), (40, 4, 128), (70, 4, 64), (36, 2, 256)])
def test_windows_around_tiles(window, n, hq, D):
    run_case(2, n, hq, 1, D, [300, 64], torch.bfloat16, window=window, kind="chain")


@pytest.mark.gpu
@pytest.mark.parametrize("length", [0, 1, 15, 16, 63, 64, 65, 127, 128, 129, 257])
@pytest.mark.parametrize("n,hq,D", [(1, 4, 64), (1, 2, 256), (40, 4, 128), (300, 1, 64)])
def test_lengths_around_tiles(length, n, hq, D):
    run_case(1, n, hq, 1, D, [length], torch.float16, cap=20.0, bias=True, window=50, kind="chain")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["chain", "star", "roots", "padded", "tree"])
@pytest.mark.parametrize("n,g", [(2, 1), (17, 3), (64, 4), (65, 2), (129, 1)])
def test_trees_stand_at_their_depths(kind, n, g):
    run_case(2, n, 2 * g, 2, 64, [70, 3], torch.bfloat16, kind=kind, tw=True, bias=True, window=6)
    run_case(2, n, 2 * g, 2, 64, [70, 3], torch.bfloat16, kind=kind, window=3, cap=8.0)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [8, 40, 80, 112, 200])
def test_head_sizes(D):
    run_case(2, 1, 6, 2, D, [50, 133], torch.float16, cap=10.0, window=60)
    run_case(2, 21, 6, 2, D, [50, 133], torch.bfloat16, bias=True, window=60)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", [8, 9, 16, 17, 24, 25, 32, 33])
def test_rows_where_the_kernels_change(rows, D):
    run_case(2, rows, 2, 2, D, [2500, 70], torch.float16, layout="pool", page=16, cap=15.0, bias=True, window=1500)


@pytest.mark.gpu
def test_long_and_ragged():
    run_case(4, 1, 4, 1, 64, [20000, 0, 777, 5], torch.bfloat16, layout="pool", page=16, cap=15.0, bias=True)
    run_case(4, 1, 4, 1, 64, [20000, 0, 777, 5], torch.bfloat16, layout="pool", page=16, window=3001)
    run_case(2, 36, 2, 1, 64, [9000, 1234], torch.bfloat16, layout="pool", page=16, cap=15.0, window=2000)
    run_case(1, 260, 2, 1, 128, [900], torch.bfloat16, kind="chain", window=300, bias=True)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 60, 129, 333, 900])
@pytest.mark.parametrize("n,g,D,lens", [(500, 3, 64, [700]), (450, 4, 128, [300, 0]), (400, 2, 256, [130])])
def test_windows_that_leave_tiles_behind(window, n, g, D, lens):
    """Chunks longer than the window: later blocks of rows see neither the cache nor the first new tokens."""
    run_case(len(lens), n, g, 1, D, lens, torch.bfloat16, kind="chain", window=window, weights=False, cap=30.0, bias=window == 60)


@pytest.mark.gpu
@pytest.mark.parametrize("n,g,D", [(1, 4, 128), (40, 4, 128), (40, 2, 256)])
def test_saturated_caps(n, g, D):
    # scores far past the cap at either end, and maxima that move along the keys
    run_case(1, n, g, 1, D, [700], torch.bfloat16, cap=3.0, sharp=30.0)


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [2e-3, 200.0, 1e4, 1e9, 1e30])
@pytest.mark.parametrize("n,g,D", [(1, 4, 128), (4, 4, 64), (40, 4, 128), (20, 4, 256)])
def test_caps_of_any_size(cap, n, g, D):
    # far above the scores a cap changes nothing, and costs no precision; far below, it is all that is left
    run_case(1, n, g, 1, D, [300], torch.bfloat16, cap=cap)


@pytest.mark.gpu
@pytest.mark.parametrize("n,g,D", [(6, 2, 64), (12, 1, 128), (40, 4, 128), (20, 4, 256)])
def test_nan_and_inf_past_the_windows_edge_stay_with_their_rows(n, g, D):
    """A value that is not finite where the window's edge passes reaches the rows that still see it only."""
    from voom_b200.runtime import kv_attention as kva

    L, window = 300, 150
    qkv, k, v = inputs(1, n, g, 1, D, [L], torch.bfloat16)
    bad = L + 2 - window  # seen by the first two rows
    far = L + n - window  # past the edge, in its tile: seen by all
    late = n - 1
    d = qkv.cuda()
    view = place(k, v, [L], "whole", 0)
    view.v[0, 0, bad, 0] = math.nan
    view.v[0, 0, bad, 1] = math.inf
    view.v[0, 0, far, 2] = math.inf
    d[0, late, g + 1, 3] = math.nan  # the last token's own value
    out = kva.tree_attention(d[:, :, :g], d[:, :, g:g + 1], d[:, :, g + 1:], kva.DraftTree.chain(1, n, "cuda"), view,
                             window=window, cap=30.0)[0].float().cpu()
    par = parents_of("chain", n)
    o, _, _ = od.scored_attention(qkv[0, :, :g], qkv[0, :, g:g + 1], qkv[0, :, g + 1:], oa.tree_sees(par), oa.tree_depth(par),
                                  k[0], v[0], D ** -0.5, window=window, cap=30.0)
    tol = 2 * STEP[torch.bfloat16] * float(v.abs().max() + 1)
    for i in range(n):
        assert bool((out[i, :, 2] == math.inf).all()), i
        assert bool(out[i, :, 3].isnan().all()) == (i == late), i
        if i < 2:
            assert bool(out[i, :, 0].isnan().all()) and bool((out[i, :, 1] == math.inf).all()), i
        else:
            check(out[i, :, :2], o[i, :, :2], tol, i)
        check(out[i, :, 4:], o[i, :, 4:], tol, i)


@pytest.mark.gpu
def test_infinite_scores_take_the_caps_ends():
    from voom_b200.runtime import kv_attention as kva

    for n in (1, 40):
        qkv, k, v = inputs(1, n, 4, 1, 64, [50], torch.bfloat16)
        d = qkv.cuda()
        d[:, :, :4] = d[:, :, :4].abs()
        view = place(k, v, [50], "whole", 0)
        view.k[0, 0, 7] = math.inf  # tanh(inf) = 1, tanh(-inf) = -1
        view.k[0, 0, 9] = -math.inf
        _, lse = kva.tree_attention(d[:, :, :4], d[:, :, 4:5], d[:, :, 5:], kva.DraftTree.chain(1, n, "cuda"), view, cap=4.0,
                                    return_lse=True)
        kk = k[0].clone()
        kk[0, 7], kk[0, 9] = 1e4, -1e4
        par = parents_of("chain", n)
        _, want, _ = od.scored_attention(qkv[0, :, :4].abs(), qkv[0, :, 4:5], qkv[0, :, 5:], oa.tree_sees(par),
                                         oa.tree_depth(par), kk, v[0], 64 ** -0.5, cap=4.0)
        check(lse[0], want, 3e-5, n)


@pytest.mark.gpu
def test_neutral_settings_and_repeats():
    """A window past everything changes no value by more than rounding; calls repeat bit for bit, in a graph too."""
    from voom_b200.runtime import kv_attention as kva

    for n, hq in ((1, 8), (40, 8)):
        qkv, k, v = inputs(2, n, hq, 2, 128, [5000, 3000], torch.bfloat16)
        d = qkv.cuda()
        view = place(k, v, [5000, 3000], "pool", 16)
        tree = kva.DraftTree.chain(2, n, "cuda")
        args = (d[:, :, :hq], d[:, :, hq:hq + 2], d[:, :, hq + 2:], tree, view)
        base, base_lse = kva.tree_attention(*args, return_lse=True)
        wide, wide_lse = kva.tree_attention(*args, return_lse=True, window=2 ** 31 - 1, slopes=torch.zeros(hq, device="cuda"))
        check(wide_lse, base_lse.double().cpu(), 3e-5, "lse")
        check(wide, base.double().cpu(), 2 * STEP[torch.bfloat16] * float(v.abs().max()), "out")
        assert torch.equal(kva.tree_attention(*args, window=2 ** 40), base)  # no window at all
        slopes = slopes_of(hq).cuda()
        kw = dict(cap=20.0, slopes=slopes, window=1500)
        w = torch.zeros((2, 2, view.max_len + n), device="cuda")
        first = kva.tree_attention(*args, weights=w, **kw)
        first_w = w.clone()
        for stream in (None, torch.cuda.Stream()):
            w.zero_()
            torch.cuda.synchronize()
            again = kva.tree_attention(*args, weights=w, stream=stream, **kw)
            torch.cuda.synchronize()
            assert torch.equal(again, first) and torch.equal(w, first_w)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = kva.tree_attention(*args, weights=w, **kw)
        w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first) and torch.equal(w, first_w)


@pytest.mark.gpu
def test_refusals():
    from voom_b200.runtime import kv_attention as kva

    qkv, k, v = inputs(1, 1, 4, 2, 64, [10], torch.bfloat16)
    d = qkv.cuda()
    view = place(k, v, [10], "whole", 0)
    args = (d[:, :, :4], d[:, :, 4:6], d[:, :, 6:], kva.DraftTree.chain(1, 1, "cuda"), view)
    for cap in (0.0, -1.0, 1e-12, math.nan, math.inf):
        with pytest.raises(ValueError, match="cap"):
            kva.tree_attention(*args, cap=cap)
    for window in (0, -3):
        with pytest.raises(ValueError, match="window"):
            kva.tree_attention(*args, window=window)
    s = slopes_of(4)
    for slopes in (s, s[:2].cuda(), s.double().cuda(), torch.zeros(8, device="cuda")[::2], s.cuda()[None]):
        with pytest.raises(ValueError, match="slopes"):
            kva.tree_attention(*args, slopes=slopes)


def test_c_entry_refuses(built_lib):
    import ctypes

    from voom_b200._lib import VOOM_E_CAPACITY, VOOM_E_INVALID_ARG, KvViewStruct, TreeAttentionArgs

    c = KvViewStruct()
    c.k = c.v = c.len = 1 << 30
    c.k_page = c.k_head = c.v_page = c.v_head = 64 * 64
    c.k_pos = c.v_pos = 64
    c.B, c.hk, c.D, c.page, c.max_len = 2, 2, 64, 64, 64

    def attn(**kw):
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
        return built_lib.voom_tree_attention(ctypes.byref(c), ctypes.byref(a), None, 0, None)

    assert attn() == VOOM_E_CAPACITY  # goes on to its scratch
    assert attn(cap=1.0, window=3, slopes=1 << 25) == VOOM_E_CAPACITY
    for bad in (dict(cap=-1.0), dict(cap=1e-42), dict(cap=math.nan), dict(cap=math.inf), dict(mask=1 << 26, window=3),
                dict(mask=1 << 26, slopes=1 << 25)):
        assert attn(**bad) == VOOM_E_INVALID_ARG, bad
    assert attn(mask=1 << 26, depth=1 << 27, window=3) == VOOM_E_CAPACITY


def old_layout(a):
    """The fields that callers built before slopes, caps and windows pass, and what may lie behind them in memory."""
    from voom_b200._lib import TreeAttentionArgs

    n = TreeAttentionArgs.slopes.offset
    raw = bytearray(bytes(a)[:n]) + bytearray(b"\xff" * 64)
    raw[TreeAttentionArgs.size.offset:n] = bytes(4)  # padding then
    return bytes(raw)


def test_callers_of_the_shorter_structure(built_lib):
    import ctypes

    from voom_b200._lib import VOOM_E_CAPACITY, VOOM_E_INVALID_ARG, KvViewStruct, TreeAttentionArgs

    names = [f[0] for f in TreeAttentionArgs._fields_]
    assert names[:10] == "q kn vn out lse mask weights token_weight status q_b".split() and names[-5:] == "size slopes depth cap window".split()
    assert TreeAttentionArgs.slopes.offset == 9 * 8 + 14 * 8 + 16
    c = KvViewStruct()
    c.k = c.v = c.len = 1 << 30
    c.k_page = c.k_head = c.v_page = c.v_head = 64 * 64
    c.k_pos = c.v_pos = 64
    c.B, c.hk, c.D, c.page, c.max_len = 2, 2, 64, 64, 64
    a = TreeAttentionArgs()
    a.q, a.kn, a.vn, a.out, a.mask, a.weights = 1 << 20, 1 << 21, 1 << 22, 1 << 23, 1 << 26, 1 << 24
    a.n, a.hq, a.scale = 3, 4, 0.125
    a.q_h = a.kn_h = a.vn_h = a.o_h = 64
    a.q_t = a.o_t = 4 * 64
    a.kn_t = a.vn_t = 2 * 64
    a.q_b = a.o_b = 3 * 4 * 64
    a.kn_b = a.vn_b = 3 * 2 * 64
    a.w_b, a.w_h = 2 * 80, 80
    raw = old_layout(a)
    assert built_lib.voom_tree_attention(ctypes.byref(c), raw, None, 0, None) == VOOM_E_CAPACITY
    assert built_lib.voom_tree_attention_scratch_bytes(ctypes.byref(c), raw) == \
        built_lib.voom_tree_attention_scratch_bytes(ctypes.byref(c), ctypes.byref(a)) > 0
    a.window = 3  # the longer one: its window is seen, and wants depths beside the mask
    assert built_lib.voom_tree_attention(ctypes.byref(c), ctypes.byref(a), None, 0, None) == VOOM_E_INVALID_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40])
def test_a_call_with_the_shorter_structure(n):
    from voom_b200 import _device
    from voom_b200._lib import TreeAttentionArgs, load
    from voom_b200.runtime import kv_attention as kva

    qkv, k, v = inputs(1, n, 4, 2, 64, [300], torch.float16)
    d = qkv.cuda()
    view = place(k, v, [300], "pool", 16)
    q, kn, vn = d[:, :, :4], d[:, :, 4:6], d[:, :, 6:]
    want = kva.tree_attention(q, kn, vn, kva.DraftTree.chain(1, n, "cuda"), view)
    out = torch.zeros_like(want)
    a = TreeAttentionArgs()
    a.q, a.kn, a.vn, a.out = (x.data_ptr() for x in (q, kn, vn, out))
    for name, x in (("q", q), ("kn", kn), ("vn", vn), ("o", out)):
        for i, s in enumerate("bth"):
            setattr(a, f"{name}_{s}", x.stride(i))
    a.n, a.hq, a.scale = n, 4, 64 ** -0.5
    raw = old_layout(a)
    lib = load()
    ws = torch.empty(lib.voom_tree_attention_scratch_bytes(view.packed, raw), dtype=torch.uint8, device="cuda")
    rc = lib.voom_tree_attention(view.packed, raw, ws.data_ptr(), ws.numel(), _device.raw_stream(view.index))
    torch.cuda.synchronize()
    assert rc == 0 and torch.equal(out, want)
