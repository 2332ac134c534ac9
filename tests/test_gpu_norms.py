"""Norms over many tensors, clipping and norm-bounded averages on the GPU, against their definitions in 64 bits
(norms_oracle.py states how far a correct result may be off).  Run on the MI355X: -m gpu."""
import copy
import math
import threading
from types import SimpleNamespace

import numpy as np
import pytest
import torch
from torch import nn

import norms_oracle as no

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "f64": torch.float64}
INF = math.inf


@pytest.fixture(scope="module", autouse=True)
def _native():
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    from accdfl_amd import _lib

    assert _lib.lib().build_id == _lib.source_build_id()
    assert _lib.walk_module() is not None
    yield


def _rand(shape, dtype="f32", scale=1.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(DT[dtype]).cuda()


def _list(sizes, dtype="f32", scale=1.0, seed=0):
    return [_rand(n, dtype, scale, seed * 1000 + i) for i, n in enumerate(sizes)]


SIZES = [[1], [7], [0], [3, 0, 5], [4095, 4096, 4097], [100_003], [1] * 191, [2, 70_001, 9, 16_384, 1]]


# --------------------------------------------------------------------------------------------------- global norm
@pytest.mark.parametrize("p", [2.0, 1.0, INF])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "%dx%d" % (len(s), max(s)))
def test_global_norm(sizes, dtype, p):
    from accdfl_amd.core.norms import global_norm

    ts = _list(sizes, dtype, 0.3, seed=len(sizes))
    got = global_norm(ts, norm_type=p)
    assert got.dtype == (torch.float64 if dtype == "f64" else torch.float32) and got.shape == () and got.is_cuda
    no.assert_norm(got, no.norm(ts, p), sum(sizes))


@pytest.mark.parametrize("count", [140, 141, 190, 191, 380, 1000])
def test_global_norm_of_more_tensors_than_one_launch_takes(count):
    from accdfl_amd.core.norms import clip_global_norm, global_norm

    ts = _list([1 + i * 37 % 5000 for i in range(count)], "bf16", 0.1, seed=3)
    n = sum(t.numel() for t in ts)
    no.assert_norm(global_norm(ts), no.norm(ts), n)
    outs, norm = clip_global_norm(ts, 0.5)
    want, wn = no.clip(ts, 0.5)
    no.assert_norm(norm, wn, n)
    for o, w in zip(outs, want):
        no.assert_close(o, w, n)


def test_global_norm_of_mixed_types():
    from accdfl_amd.core.norms import clip_global_norm_, global_norm

    ts = [_rand(5001, d, 0.5, i) for i, d in enumerate(["bf16", "f32", "f16", "f32", "bf16"])]
    got = global_norm(ts)
    assert got.dtype == torch.float32
    no.assert_norm(got, no.norm(ts), 25_005)
    ts.append(_rand(33, "f64", 0.5, 9))
    got = global_norm(ts)
    assert got.dtype == torch.float64
    want, wn = no.clip(ts, 3.0)
    no.assert_norm(got, wn, 25_038)
    no.assert_norm(clip_global_norm_(ts, 3.0), wn, 25_038)
    for t, w in zip(ts, want):
        no.assert_close(t, w, 25_038)


def test_global_norm_of_nothing():
    from accdfl_amd.core.norms import clip_global_norm, clip_global_norm_, clip_grad_norm_, global_norm

    assert float(global_norm([])) == 0.0 and float(clip_global_norm_([], 1.0)) == 0.0
    assert clip_global_norm([], 1.0)[0] == []
    assert float(clip_grad_norm_(nn.Linear(3, 3).cuda(), 1.0)) == 0.0
    empty = [torch.empty(0, device="cuda"), torch.empty(3, 0, device="cuda")]
    assert float(global_norm(empty)) == 0.0
    outs, n = clip_global_norm(empty, 1.0)
    assert float(n) == 0.0 and [o.shape for o in outs] == [(0,), (3, 0)]


@pytest.mark.parametrize("value", [3e38, 1e-38, 1e-45, 2e19])
def test_norm_does_not_overflow_or_underflow(value):
    from accdfl_amd.core.norms import global_norm

    ts = [torch.full((1000,), value / 64, device="cuda"), torch.full((24,), value / 64, device="cuda")]
    no.assert_norm(global_norm(ts), no.norm(ts), 1024)
    no.assert_norm(global_norm([t.bfloat16() for t in ts]), no.norm([t.bfloat16() for t in ts]), 1024)


@pytest.mark.parametrize("p", [2.0, 1.0, INF])
@pytest.mark.parametrize("bad", [math.nan, INF, -INF])
@pytest.mark.parametrize("where", [0, 4095, 70_000])
def test_nonfinite_norms(p, bad, where):
    from accdfl_amd.core.norms import clip_global_norm_, global_norm

    ts = [_rand(9), _rand(70_001, seed=1)]
    ts[1][where] = bad
    want = no.norm(ts, p)
    no.assert_norm(global_norm(ts, p), want, 70_010)
    with pytest.raises(RuntimeError, match="not finite"):
        global_norm(ts, p, error_if_nonfinite=True)
    before = [t.clone() for t in ts]
    with pytest.raises(RuntimeError, match="not finite"):
        clip_global_norm_(ts, 1.0, p, error_if_nonfinite=True)
    assert all(torch.equal(a, b) or bool(torch.isnan(a).any()) for a, b in zip(ts, before))
    expect, _ = no.clip(before, 1.0, p)
    clip_global_norm_(ts, 1.0, p)
    for t, w in zip(ts, expect):
        no.assert_close(t, w, 70_010)


def test_infinity_norm_keeps_a_nan_beside_an_infinity():
    from accdfl_amd.core.norms import global_norm

    for order in ((math.nan, INF), (INF, math.nan)):
        t = torch.zeros(100_000, device="cuda")
        t[17], t[90_001] = order
        assert math.isnan(float(global_norm([t], INF)))


# ------------------------------------------------------------------------------------------------------ clipping
@pytest.mark.parametrize("p", [2.0, 1.0, INF])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("max_norm", [0.0, 0.37, 1e9, INF])
def test_clip(dtype, p, max_norm):
    from accdfl_amd.core.norms import clip_global_norm, clip_global_norm_

    sizes = [1, 4097, 0, 20_011]
    ts = _list(sizes, dtype, 0.7, seed=5)
    before = [t.clone() for t in ts]
    want, wn = no.clip(ts, max_norm, p)
    outs, n = clip_global_norm(ts, max_norm, norm_type=p)
    no.assert_norm(n, wn, sum(sizes))
    for t, b, o, w in zip(ts, before, outs, want):
        assert torch.equal(t, b) and o.dtype == t.dtype and o.data_ptr() != t.data_ptr() or t.numel() == 0
        no.assert_close(o, w, sum(sizes))
    no.assert_norm(clip_global_norm_(ts, max_norm, norm_type=p), wn, sum(sizes))
    for t, o, b in zip(ts, outs, before):
        assert torch.equal(t, o)  # in place and out of place are the same bits
        if max_norm >= 1e9:
            assert torch.equal(t, b)


@pytest.mark.parametrize("dtype", list(DT))
def test_clip_rounds_once(dtype):
    """Products at a power of two below the values are exact; the others within half a step of x * ratio in 64 bits."""
    from accdfl_amd.core.norms import clip_global_norm

    t = _rand(65_537, dtype, 1.0, 2)
    for bound in (1e-3, 0.77, 100.0):
        (out,), _ = clip_global_norm([t], bound)
        no.assert_close(out, no.clip([t], bound)[0][0], 65_537)


def test_clip_into_subnormals():
    from accdfl_amd.core.norms import clip_global_norm

    for dtype, scale in (("f16", 1e-3), ("bf16", 1e-30), ("f32", 1e-30)):
        t = _rand(5000, dtype, scale, 4)
        bound = float(no.norm([t])) * {"f16": 1e-3, "bf16": 1e-9, "f32": 1e-9}[dtype]
        (out,), _ = clip_global_norm([t.double().to(DT[dtype])], bound)
        # eps counts for nothing here only beside norms far above it: take the ratio as it is defined
        no.assert_close(out, no.clip([t], bound)[0][0], 5000)


@pytest.mark.parametrize("dtype", ["bf16", "f32", "f64"])
@pytest.mark.parametrize("start", [1, 3])
def test_tensors_that_start_anywhere(dtype, start):
    """Views into one buffer, back to back from an odd element on; what lies around them stays as it was."""
    from accdfl_amd.core.norms import clip_global_norm, clip_global_norm_, global_norm

    sizes = [5, 4099, 1, 2050, 333]
    total = sum(sizes)
    buf = _rand(total + start + 7, dtype, 0.5, 6)
    views = list(torch.split(buf[start:start + total], sizes))
    n = no.norm(views)
    no.assert_norm(global_norm(views), n, total)
    sent = torch.full_like(buf, 7.0)
    outs = list(torch.split(sent[start + 2:start + 2 + total], sizes))  # another alignment than the inputs'
    want, _ = no.clip(views, 0.4)
    clip_global_norm(views, 0.4, outs=outs)
    for o, w in zip(outs, want):
        no.assert_close(o, w, total)
    assert bool((sent[:start + 2] == 7).all()) and bool((sent[start + 2 + total:] == 7).all())
    edge = buf[:start].clone(), buf[start + total:].clone()
    clip_global_norm_(views, 0.4)
    for v, w in zip(views, want):
        no.assert_close(v, w, total)
    assert torch.equal(buf[:start], edge[0]) and torch.equal(buf[start + total:], edge[1])


def test_axes_in_any_order_and_views_with_gaps():
    from accdfl_amd.core.norms import clip_global_norm, clip_global_norm_, global_norm

    conv = _rand((8, 4, 3, 3), "f32", 0.5, 7).to(memory_format=torch.channels_last)
    base = _rand((50, 40), "f32", 0.5, 8)
    gaps, spread = base[:, :13], _rand((30, 1), "f32", 0.5, 9).expand(30, 20)
    lists = [conv, base.t()[20:], gaps, spread, _rand((), "f32", 1.0, 10), conv[:, 1]]
    n = sum(t.numel() for t in lists)
    no.assert_norm(global_norm(lists), no.norm(lists), n)
    outs, norm = clip_global_norm(lists, 0.9)
    want, wn = no.clip(lists, 0.9)
    no.assert_norm(norm, wn, n)
    for o, w, t in zip(outs, want, lists):
        assert o.shape == t.shape
        no.assert_close(o, w, n)
    # in place: views with gaps are written, the gaps are not; an expanded tensor is refused
    with pytest.raises(ValueError, match="share memory"):
        clip_global_norm_([spread], 0.1)
    rest = base[:, 13:].clone()
    want, _ = no.clip([gaps, conv], 0.1)
    clip_global_norm_([gaps, conv], 0.1)
    no.assert_close(gaps, want[0], n)
    no.assert_close(conv, want[1], n)
    assert torch.equal(base[:, 13:], rest)


def test_overlaps_are_refused():
    from accdfl_amd import _lib
    from accdfl_amd.core.norms import clip_global_norm, clip_global_norm_

    t = _rand(100)
    before = t.clone()
    for bad in ([t, t], [t[:60], t[50:]]):
        with pytest.raises(_lib.DlaggError, match="overlap"):
            clip_global_norm_(bad, 0.1)
    with pytest.raises(_lib.DlaggError, match="overlap"):
        clip_global_norm([t[:50]], 0.1, outs=[t[1:51]])
    assert torch.equal(t, before)
    # the same tensor twice counts twice where nothing overlaps what is written
    outs, n = clip_global_norm([t, t], 0.1)
    no.assert_norm(n, no.norm([t, t]), 200)
    assert torch.equal(outs[0], outs[1])


def test_wrong_lists_are_refused():
    from accdfl_amd.core import norms

    t = _rand(10)
    with pytest.raises(ValueError, match="cpu"):
        norms.global_norm([t, torch.zeros(3)])
    with pytest.raises(ValueError):
        norms.global_norm([torch.zeros(3)])
    with pytest.raises(TypeError):
        norms.global_norm([torch.zeros(3, dtype=torch.int32, device="cuda")])
    with pytest.raises(TypeError):
        norms.global_norm([torch.zeros(3, dtype=torch.complex64, device="cuda")])
    with pytest.raises(TypeError, match="strided"):
        norms.global_norm([torch.eye(3, device="cuda").to_sparse()])
    with pytest.raises(TypeError, match="not a tensor"):
        norms.global_norm([t, 3.0])
    with pytest.raises(ValueError, match="outs"):
        norms.clip_global_norm([t], 1.0, outs=[])
    with pytest.raises(ValueError, match="outs"):
        norms.clip_global_norm([t], 1.0, outs=[torch.zeros(11, device="cuda")])
    with pytest.raises(ValueError, match="outs"):
        norms.clip_global_norm([t], 1.0, outs=[torch.zeros(10, device="cuda", dtype=torch.float16)])
    with pytest.raises(ValueError, match="model 1"):
        norms.update_norms([[t], [t, t]], [t])
    with pytest.raises(ValueError, match="model 0"):
        norms.update_norms([[t.half()]], [t])
    with pytest.raises(ValueError, match="peer 1"):
        norms.wsum_bounded_multi([[t], [t[:5]]], [0.5, 0.5], [t], 1.0, [torch.empty_like(t)])
    with pytest.raises(ValueError, match="sq_norms"):
        norms.wsum_bounded([t], [1.0], t, 1.0, sq_norms=torch.zeros(1, device="cuda"))


def test_clip_grad_norm_is_torchs_contract():
    from accdfl_amd.core.norms import clip_grad_norm_

    torch.manual_seed(0)
    model = nn.Sequential(nn.Conv2d(3, 8, 3), nn.Flatten(), nn.Linear(8 * 36, 11), nn.Linear(11, 5, bias=False)).cuda()
    model(torch.randn(4, 3, 8, 8, device="cuda")).square().sum().backward()
    model[3].weight.grad = None
    twin = copy.deepcopy(model)
    for p, q in zip(model.parameters(), twin.parameters()):
        q.grad = None if p.grad is None else p.grad.clone()
    versions = [p.grad._version for p in model.parameters() if p.grad is not None]
    want, wn = no.clip([p.grad for p in twin.parameters() if p.grad is not None], 0.5)
    got = clip_grad_norm_(model.parameters(), 0.5)
    n = sum(w.numel() for w in want)
    no.assert_norm(got, wn, n)
    stock = torch.nn.utils.clip_grad_norm_(twin.parameters(), 0.5)
    assert abs(float(stock) - float(got)) <= 1e-5 * float(got)
    for p, q, w in zip([p for p in model.parameters() if p.grad is not None],
                       [p for p in twin.parameters() if p.grad is not None], want):
        no.assert_close(p.grad, w, n)
        assert torch.allclose(p.grad, q.grad, rtol=2e-5, atol=0)
    assert all(p.grad._version > v for p, v in zip([p for p in model.parameters() if p.grad is not None], versions))
    assert model[3].weight.grad is None
    before = [p.grad.clone() for p in model.parameters() if p.grad is not None]
    clip_grad_norm_(model, 1e6)  # a module; nothing to clip
    assert all(torch.equal(p.grad, b) for p, b in zip([p for p in model.parameters() if p.grad is not None], before))


# ----------------------------------------------------------------------------------------- peers around a centre
def _round(n, sizes, dtype, seed=0, scale=0.02):
    center = _list(sizes, dtype, 0.5, seed=seed + 100)
    models = [[(c.double() + _rand(c.shape, "f64", scale * (1 + k % 4), seed * 7919 + 31 * k + i).view_as(c)).to(c.dtype)
               for i, c in enumerate(center)] for k in range(n)]
    weights = [float(w) for w in np.random.default_rng(n).dirichlet(np.ones(n))]
    return center, models, weights


PEERS = [1, 2, 3, 5, 7, 8, 9, 16, 23, 64, 130]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n", PEERS)
def test_update_norms(n, dtype):
    from accdfl_amd.core.norms import update_norms

    sizes = [1, 1025, 0, 6007]
    center, models, _ = _round(n, sizes, dtype)
    got = update_norms(models, center)
    assert got.shape == (n,) and got.dtype == (torch.float64 if dtype == "f64" else torch.float32)
    want = no.update_norms(models, center)
    no.assert_norm(got, want, sum(sizes))
    sq = update_norms(models, center, squared=True)
    assert sq.dtype == torch.float64
    np.testing.assert_allclose(sq.sqrt().cpu().numpy(), want, rtol=2.0 ** -53 * (sum(sizes) + 16))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n", PEERS)
def test_wsum_bounded_multi(n, dtype):
    from accdfl_amd.core.norms import wsum_bounded_multi

    sizes = [1, 1025, 0, 6007, 4]
    center, models, weights = _round(n, sizes, dtype)
    norms = no.update_norms(models, center)
    bound = sorted(norms)[n // 2] * 0.9
    outs = [torch.full_like(c, 9.0) for c in center]
    got = wsum_bounded_multi(models, weights, center, bound, outs)
    want, wn, added = no.bounded(models, weights, center, bound)
    no.assert_norm(got, wn, sum(sizes))
    for o, w, a in zip(outs, want, added):
        no.assert_close(o, w, sum(sizes) + n, a)


@pytest.mark.parametrize("numel", [1, 2, 1023, 1024, 1025, 300_007])
@pytest.mark.parametrize("dtype", list(DT))
def test_wsum_bounded_flat(numel, dtype):
    from accdfl_amd.core.norms import wsum_bounded

    (center,), models, weights = _round(6, [numel], dtype, seed=2)
    peers = [m[0] for m in models]
    for bound in (0.0, 0.02 * math.sqrt(numel), INF):
        out, norms = wsum_bounded(peers, weights, center, bound)
        want, wn, added = no.bounded(models, weights, [center], bound)
        no.assert_norm(norms, wn, numel)
        no.assert_close(out, want[0], numel + 6, added[0])
        if bound == 0.0:
            assert torch.equal(out, center)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_broken_peers_add_nothing(dtype):
    from accdfl_amd.core.norms import wsum_bounded

    (center,), models, weights = _round(11, [9001], dtype, seed=4)
    peers = [m[0] for m in models]
    peers[0][9000] = math.nan
    peers[4][0] = INF
    peers[10][123] = -INF
    out, norms = wsum_bounded(peers, weights, center, 1.0)
    want, wn, added = no.bounded([[p] for p in peers], weights, [center], 1.0)
    no.assert_norm(norms, wn, 9001)
    assert math.isnan(float(norms[0])) and float(norms[4]) == INF and float(norms[10]) == INF
    assert bool(torch.isfinite(out).all())
    no.assert_close(out, want[0], 9100, added[0])
    out, _ = wsum_bounded([torch.full_like(center, math.nan)] * 3, [0.2] * 3, center, 1.0)
    assert torch.equal(out, center)
    # a broken centre: every update is broken, the centre stays
    center[5] = math.nan
    out, norms = wsum_bounded(peers[1:4], weights[1:4], center, 1.0)
    assert bool(torch.isnan(norms).all()) and math.isnan(float(out[5]))
    assert torch.equal(out[:5], center[:5]) and torch.equal(out[6:], center[6:])


def test_extreme_updates():
    """Differences that overflow float32, and updates whose squares underflow it."""
    from accdfl_amd.core.norms import wsum_bounded

    center = torch.full((1000,), -3e38, device="cuda")
    peer = torch.full((1000,), 3e38, device="cuda")
    out, norms = wsum_bounded([peer], [0.25], center, INF)
    want, wn, added = no.bounded([[peer]], [0.25], [center], INF)
    assert float(norms[0]) == INF and wn[0] > 1e40  # 6e38 * sqrt(1000) is beyond float32, not beyond the sums
    no.assert_close(out, want[0], 1000, added[0])
    center = torch.zeros(1000, device="cuda")
    peer = torch.full((1000,), 1e-30, device="cuda")
    out, norms = wsum_bounded([peer], [1.0], center, 1e-30)
    want, wn, added = no.bounded([[peer]], [1.0], [center], 1e-30)
    no.assert_norm(norms, wn, 1000)
    no.assert_close(out, want[0], 1000, added[0])


def test_weights_of_zero_negative_and_beyond_one():
    from accdfl_amd.core.norms import wsum_bounded

    (center,), models, _ = _round(4, [5003], "f32", seed=6)
    weights = [0.0, -0.5, 3.0, 1.0]
    out, _ = wsum_bounded([m[0] for m in models], weights, center, 1.5)
    want, _, added = no.bounded(models, weights, [center], 1.5)
    no.assert_close(out, want[0], 5100, added[0])


def test_without_a_bound_it_is_the_weighted_average():
    from accdfl_amd.core import wsum
    from accdfl_amd.core.norms import wsum_bounded

    (center,), models, weights = _round(8, [40_001], "f32", seed=8)
    peers = [m[0] for m in models]
    out, _ = wsum_bounded(peers, weights, center, INF)
    avg = wsum.wsum(peers, weights)
    mag = sum(w * p.double().abs() for w, p in zip(weights, peers)) + center.double().abs()
    # FedAvg rounds 8 products and 8 sums; sum of the weights is 1 within 8 * 2^-53
    assert bool(((out.double() - avg.double()).abs() <= 17 * 2.0 ** -24 * mag).all())


def test_out_may_be_the_centre_or_a_peer():
    from accdfl_amd import _lib
    from accdfl_amd.core.norms import wsum_bounded

    for which in ("center", "peer"):
        (center,), models, weights = _round(3, [70_001], "bf16", seed=9)
        peers = [m[0] for m in models]
        want, _ = wsum_bounded(peers, weights, center, 2.0)
        out = center if which == "center" else peers[1]
        version = out._version
        got, _ = wsum_bounded(peers, weights, center, 2.0, out=out)
        assert got is out and torch.equal(got, want) and out._version > version
    with pytest.raises(_lib.DlaggError, match="overlap"):
        wsum_bounded([center[:-1], center[:-1]], [0.5, 0.5], center[:-1], 1.0, out=center[1:])
    # a client's own update, bounded before it is sent
    (center,), models, _ = _round(1, [5001], "f32", seed=10)
    model = models[0][0]
    want, wn, added = no.bounded(models, [1.0], [center], 0.5)
    wsum_bounded([model], [1.0], center, 0.5, out=model)
    no.assert_close(model, want[0], 5001, added[0])
    assert abs(no.norm([model.double() - center.double()]) - 0.5) <= 1e-4


def test_peers_in_other_element_orders():
    from accdfl_amd.core.norms import update_norms, wsum_bounded

    center = _rand((40, 30), "f32", 0.5, 1)
    a = (center + _rand((40, 30), "f32", 0.1, 2)).t().contiguous().t()
    wide = torch.zeros(40, 60, device="cuda")
    wide[:, ::2] = center + _rand((40, 30), "f32", 0.2, 3)
    peers = [a, wide[:, ::2], center.clone()]
    no.assert_norm(update_norms([[p] for p in peers], [center]), no.update_norms([[p] for p in peers], [center]), 1200)
    want, _, added = no.bounded([[p] for p in peers], [0.3, 0.3, 0.4], [center], 1.0)
    for out in (None, torch.empty(30, 40, device="cuda").t(), wide[:, 1::2]):
        got, _ = wsum_bounded(peers, [0.3, 0.3, 0.4], center, 1.0, out=out)
        no.assert_close(got, want[0], 1200, added[0])
    # all in one other order: read where they are
    got, _ = wsum_bounded([p.t().contiguous().t() for p in peers], [0.3, 0.3, 0.4], center.t().contiguous().t(), 1.0)
    no.assert_close(got, want[0], 1200, added[0])


def test_mixed_types_across_a_model():
    from accdfl_amd.core.norms import update_norms, wsum_bounded_multi

    rounds = [_round(5, [n], d, seed=i) for i, (n, d) in enumerate([(3001, "bf16"), (40, "f32"), (5000, "f16"), (7, "bf16")])]
    center = [r[0][0] for r in rounds]
    models = [[r[1][k][0] for r in rounds] for k in range(5)]
    weights = rounds[0][2]
    no.assert_norm(update_norms(models, center), no.update_norms(models, center), 8048)
    outs = [torch.empty_like(c) for c in center]
    wsum_bounded_multi(models, weights, center, 1.0, outs)
    want, _, added = no.bounded(models, weights, center, 1.0)
    for o, w, a in zip(outs, want, added):
        no.assert_close(o, w, 8100, a)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("numel, capacity, n", [(1, 1, 1), (5003, 8, 8), (5003, 8, 3), (300_001, 5, 5), (70_000, 40, 33)])
@pytest.mark.parametrize("own_center", [False, True])
def test_slab_rows(dtype, numel, capacity, n, own_center):
    from accdfl_amd.core.peer_slab import PeerSlab

    center, models, weights = _round(n, [numel], dtype, seed=3)
    slab = PeerSlab([(numel,)], DT[dtype], capacity)
    for m in models:
        slab.stage(m)
    c = center if own_center else models[0]
    bound = 0.03 * math.sqrt(numel)
    out, norms = slab.reduce_bounded(bound, weights, center=center if own_center else None)
    want, wn, added = no.bounded(models, weights, c, bound)
    no.assert_norm(norms, wn, numel)
    no.assert_close(out, want[0], numel + n, added[0])
    for k in range(n):
        assert torch.equal(slab.row(k), models[k][0])


def test_many_peers_and_the_largest_count():
    from accdfl_amd.core.norms import update_norms, wsum_bounded

    g = torch.Generator().manual_seed(1)
    peers = torch.randn(2048, 33, generator=g).cuda()
    center = torch.zeros(33, device="cuda")
    weights = [1.0 / 2048] * 2048
    rows = list(peers)
    no.assert_norm(update_norms(rows, center), no.update_norms([[p] for p in rows], [center]), 33)
    out, _ = wsum_bounded(rows, weights, center, 5.0)
    want, _, added = no.bounded([[p] for p in rows], weights, [center], 5.0)
    no.assert_close(out, want[0], 4096, added[0])


def test_many_tensors_of_many_peers():
    """A table of several thousand words, and tensors found by a search of two steps."""
    from accdfl_amd.core.norms import wsum_bounded_multi

    sizes = [1 + i * 7 % 90 for i in range(5000)]
    center = list(torch.split(_rand(sum(sizes), "f32", 0.5, 1), sizes))
    flats = [_rand(sum(sizes), "f32", 0.02, 10 + k) + torch.cat(center) for k in range(3)]
    models = [list(torch.split(f, sizes)) for f in flats]
    out = torch.full((sum(sizes),), 9.0, device="cuda")
    norms = wsum_bounded_multi(models, [0.2, 0.3, 0.5], center, 5.0, list(torch.split(out, sizes)))
    want, wn, added = no.bounded([[f] for f in flats], [0.2, 0.3, 0.5], [torch.cat(center)], 5.0)
    no.assert_norm(norms, wn, sum(sizes))
    no.assert_close(out, want[0], sum(sizes), added[0])


# ----------------------------------------------------------------------------------- modules, managers, a whole run
class _Net(nn.Module):
    def __init__(self, seed, dtype=torch.float32, gains=None):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        p = lambda *s, d=dtype: nn.Parameter((torch.randn(*s, generator=g) * 0.1).to(d))  # noqa: E731
        self.w = p(40, 30)
        self.gain = p(30, d=gains or dtype)
        self.inner = nn.ParameterList([p(7), p(3, 5, 2)])
        self.register_buffer("seen", torch.full((3,), float(seed)))


def _net_case(device, dtype=torch.float32, gains=None, n=5):
    models = [_Net(k + 1, dtype, gains).to(device) for k in range(n)]
    center = _Net(99, dtype, gains).to(device)
    return models, center, [0.1, 0.2, 0.3, 0.25, 0.15][:n]


def _check_module(out, models, center, weights, bound, device):
    want, _, added = no.bounded([list(m.parameters()) for m in models], weights, list(center.parameters()), bound)
    got = list(out.parameters())
    assert type(out) is type(models[0]) and len(got) == len(want)
    assert torch.equal(out.seen, models[0].seen) and out.seen.data_ptr() != models[0].seen.data_ptr()
    for o, w, a, p in zip(got, want, added, models[0].parameters()):
        assert o.device == torch.device(device) and o.requires_grad == p.requires_grad and o.dtype == p.dtype
        no.assert_close(o, w, 2000, a)


@pytest.mark.parametrize("device", ["cpu", "cuda:0"])
@pytest.mark.parametrize("dtype, gains", [(torch.float32, None), (torch.bfloat16, None), (torch.float64, None),
                                          (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("own_center", [False, True])
def test_norm_bounded_fedavg(device, dtype, gains, own_center):
    from accdfl_amd.core.gradient_aggregation.norm_bounded import NormBoundedFedAvg

    models, center, weights = _net_case(device, dtype, gains)
    before = [[p.detach().clone() for p in m.parameters()] for m in models]
    out = NormBoundedFedAvg(3.0, center if own_center else None).aggregate(models, weights)
    _check_module(out, models, center if own_center else models[0], weights, 3.0, device)
    assert all(torch.equal(p, b) for m, bs in zip(models, before) for p, b in zip(m.parameters(), bs))
    out = NormBoundedFedAvg(3.0, center).aggregate(models, None)  # uniform
    _check_module(out, models, center, [0.2] * 5, 3.0, device)


@pytest.mark.parametrize("device", ["cpu", "cuda:0"])
def test_norm_bounded_fedavg_of_channels_last_models(device):
    """Models whose parameters have another element order, all of them or one of them."""
    from accdfl_amd.core.gradient_aggregation.norm_bounded import NormBoundedFedAvg

    for orders in ((True, True, True, True), (True, False, True, False), (False, True, True, False)):
        models = []
        for k, last in enumerate(orders):
            torch.manual_seed(k)
            net = nn.Sequential(nn.Conv2d(4, 6, 3), nn.BatchNorm2d(6), nn.Conv2d(6, 5, 3, bias=False)).to(device)
            models.append(net.to(memory_format=torch.channels_last) if last else net)
        center = models.pop()
        out = NormBoundedFedAvg(1.0, center).aggregate(models, [0.2, 0.3, 0.5])
        want, _, added = no.bounded([list(m.parameters()) for m in models], [0.2, 0.3, 0.5], list(center.parameters()), 1.0)
        for o, w, a, p in zip(out.parameters(), want, added, models[0].parameters()):
            assert o.stride() == p.stride() and o.device == p.device
            no.assert_close(o, w, 1000, a)


def test_norm_bounded_fedavg_of_models_in_two_places():
    from accdfl_amd.core.gradient_aggregation.norm_bounded import NormBoundedFedAvg

    models, center, weights = _net_case("cuda:0")
    models[2] = models[2].cpu()
    _check_module(NormBoundedFedAvg(3.0, center.cpu()).aggregate(models, weights), models, center, weights, 3.0, "cuda:0")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("own_center", [False, True])
def test_norm_bounded_fedavg_of_large_cpu_models(dtype, own_center):
    """Rows beyond one page-locked buffer, tensors cut at its end, empty tensors, two calls at once."""
    from accdfl_amd.core.gradient_aggregation import norm_bounded

    def model(seed):
        g = torch.Generator().manual_seed(seed)
        return nn.ParameterList([nn.Parameter((torch.randn(s, generator=g) * 0.1).to(dtype))
                                 for s in ((3, 5), (0,), (2_000_003,), (7,), (1500, 2001), (1,))])

    models, center = [model(k) for k in range(4)], model(50)
    weights = [0.4, 0.3, 0.2, 0.1]
    c = center if own_center else models[0]
    want, _, added = no.bounded([list(m) for m in models], weights, list(c), 200.0)
    outs = [None, None]

    def work(i):
        outs[i] = norm_bounded.NormBoundedFedAvg(200.0, center if own_center else None).aggregate(models, weights)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(100)
    for out in outs:
        for o, w, a in zip(out, want, added):
            assert o.is_cpu
            no.assert_close(o, w, 5_001_530, a)
    norm_bounded.release_staging()


@pytest.mark.parametrize("with_model", [False, True])
def test_managers(with_model):
    """Both managers, the registry's order; the device manager's round runs over its staged slab rows."""
    from accdfl_amd.core import wire
    from accdfl_amd.core.gradient_aggregation import GradientAggregationMethod
    from accdfl_amd.core.model_manager import DeviceModelManager, ModelManager

    settings = SimpleNamespace(gradient_aggregation=GradientAggregationMethod.NORM_BOUNDED_FEDAVG, max_update_norm=3.0)
    models, center, weights = _net_case("cpu")
    own = center if with_model else None
    c = center if with_model else models[0]
    plain = ModelManager(own, settings)
    staged = DeviceModelManager(own, settings, capacity=2, template=_Net(5))
    wired = DeviceModelManager(own, settings, capacity=8, template=_Net(5))
    for k, m in enumerate(models):
        plain.process_incoming_trained_model(b"p%d" % k, m)
        staged.process_incoming_trained_model(b"p%d" % k, m)
        wired.process_incoming_serialized(b"p%d" % k, wire.serialize_model(m))
    for mm in (plain, staged, wired):
        _check_module(mm.aggregate_trained_models(weights), models, c, weights, 3.0, "cpu")
    back = wire.loads_state_dict(wired.aggregate_serialized(weights))
    out = copy.deepcopy(models[0])
    out.load_state_dict(back)
    _check_module(out, models, c, weights, 3.0, "cpu")


@pytest.mark.parametrize("device", ["cpu", "cuda:0"])
def test_a_round_with_local_steps(device):
    """As they are used: every client trains with clipped gradients, bounds its own update, and the round averages
    what arrives under the same bound; one client sends NaNs."""
    from accdfl_amd.core.gradient_aggregation.norm_bounded import NormBoundedFedAvg
    from accdfl_amd.core.norms import clip_grad_norm_, update_norms, wsum_bounded_multi

    torch.manual_seed(0)
    start = nn.Sequential(nn.Linear(20, 16), nn.Tanh(), nn.Linear(16, 3)).cuda()
    clients = []
    for k in range(4):
        model = copy.deepcopy(start)
        opt = torch.optim.SGD(model.parameters(), lr=1.0)
        for _ in range(3):
            opt.zero_grad()
            nn.functional.mse_loss(model(torch.randn(8, 20, device="cuda")), torch.randn(8, 3, device="cuda") * 5).backward()
            grads = [p.grad.clone() for p in model.parameters()]
            want, wn = no.clip(grads, 0.3)
            no.assert_norm(clip_grad_norm_(model.parameters(), 0.3), wn, 400)
            for p, w in zip(model.parameters(), want):
                no.assert_close(p.grad, w, 400)
            opt.step()
        clients.append(model)
    moved = [list(p.detach() for p in m.parameters()) for m in clients]
    base = [p.detach() for p in start.parameters()]
    want, wn, added = no.bounded([moved[0]], [1.0], base, 0.2)
    assert wn[0] > 0.2
    wsum_bounded_multi([moved[0]], [1.0], base, 0.2, moved[0])
    for m, w, a in zip(moved[0], want, added):
        no.assert_close(m, w, 400, a)
    with torch.no_grad():
        clients[3][0].weight[0, 0] = math.nan
    models, center = [m.to(device) for m in clients], start.to(device)
    out = NormBoundedFedAvg(0.4, center).aggregate(models, None)
    want, wn, added = no.bounded([list(m.parameters()) for m in models], [0.25] * 4, list(center.parameters()), 0.4)
    assert math.isnan(wn[3])
    for o, w, a in zip(out.parameters(), want, added):
        no.assert_close(o, w, 400, a)
    n = update_norms([out.cuda()], start.cuda())
    assert float(n) <= 0.4 * 0.75 * (1 + 1e-6)


# -------------------------------------------------------------------------- streams, threads, graphs, large offsets
def test_other_streams_and_threads():
    from accdfl_amd.core.norms import clip_global_norm, update_norms, wsum_bounded

    (center,), models, weights = _round(5, [200_003], "f32", seed=12)
    peers = [m[0] for m in models]
    want_out, want_norms = wsum_bounded(peers, weights, center, 5.0)
    want_clip = clip_global_norm(peers, 1.0)
    torch.cuda.synchronize()
    errors = []

    def work(seed):
        try:
            st = torch.cuda.Stream()
            for i in range(20):
                if (seed + i) % 2:
                    out, norms = wsum_bounded(peers, weights, center, 5.0, stream=st)
                    clipped, n = clip_global_norm(peers, 1.0, stream=st)
                else:
                    with torch.cuda.stream(st):
                        out, norms = wsum_bounded(peers, weights, center, 5.0)
                        clipped, n = clip_global_norm(peers, 1.0)
                        update_norms(peers, center)
                st.synchronize()
                assert torch.equal(out, want_out) and torch.equal(norms, want_norms)
                assert torch.equal(n, want_clip[1]) and all(torch.equal(a, b) for a, b in zip(clipped, want_clip[0]))
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(100)
    assert not errors, errors


def test_two_captured_graphs_replay_beside_eager_calls():
    from accdfl_amd.core.norms import clip_global_norm, clip_global_norm_, global_norm, update_norms, wsum_bounded_multi

    sizes = [4097, 3, 60_001]
    center, models, weights = _round(9, sizes, "f32", seed=13)
    grads = _list(sizes, "bf16", 0.5, seed=14)
    kept = [g.clone() for g in grads]
    outs, sent = [torch.zeros_like(c) for c in center], [torch.zeros_like(g) for g in grads]

    def first():
        return global_norm(grads), clip_global_norm(grads, 0.5, outs=sent)[1], clip_global_norm_(grads, 2.0)

    def second():
        return update_norms(models, center), wsum_bounded_multi(models, weights, center, 1.0, outs)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # warm up
        first(), second()
    side.synchronize()
    graphs, results = [], []
    for fn in (first, second):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            results.append(fn())
        graphs.append(g)
    for i in range(4):
        for g, k in zip(grads, kept):
            g.copy_(k * (i + 1))
        for m in models[i]:
            m.add_(0.5)
        for t in outs + sent:
            t.zero_()
        expect_clip = no.clip(grads, 0.5)
        expect_in_place = no.clip(grads, 2.0)
        expect = no.bounded(models, weights, center, 1.0)
        torch.cuda.synchronize()
        # both at once, on two streams, with eager calls of the same operators beside them
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        with torch.cuda.stream(a):
            graphs[0].replay()
        with torch.cuda.stream(b):
            graphs[1].replay()
        update_norms(models, center)
        torch.cuda.synchronize()
        n = sum(sizes)
        no.assert_norm(results[0][0], expect_clip[1], n)
        no.assert_norm(results[0][1], expect_clip[1], n)
        no.assert_norm(results[0][2], expect_clip[1], n)
        no.assert_norm(results[1][0], expect[1], n)
        no.assert_norm(results[1][1], expect[1], n)
        for s, w in zip(sent, expect_clip[0]):
            no.assert_close(s, w, n)
        for g, w in zip(grads, expect_in_place[0]):
            no.assert_close(g, w, n)
        for o, w, ad in zip(outs, expect[0], expect[2]):
            no.assert_close(o, w, n, ad)


def test_counters_are_zero_again_and_calls_without_them_agree():
    """Eager calls join in their last workgroup, captured ones in a launch of their own: the same bits."""
    from accdfl_amd.core import norms

    grads = _list([1 + i * 131 % 9000 for i in range(400)], "bf16", 0.5, seed=21)
    rounds = [_round(n, [70_003, 5], "f32", seed=n) for n in (1, 8, 9, 130)]

    def everything():
        out = [norms.global_norm(grads, p) for p in (2.0, 1.0, INF)]
        clipped, n = norms.clip_global_norm(grads, 0.5)
        out += clipped + [n]
        for center, models, weights in rounds:
            outs = [torch.empty_like(c) for c in center]
            out += [norms.update_norms(models, center), norms.wsum_bounded_multi(models, weights, center, 3.0, outs)] + outs
        return out

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        eager = [everything() for _ in range(3)]
    side.synchronize()
    for again in eager[1:]:
        assert all(torch.equal(a, b) for a, b in zip(eager[0], again))
    assert (0, side.cuda_stream) in norms._counters
    assert all(int(c.abs().max()) == 0 for c in norms._counters.values())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        captured = everything()
    for _ in range(3):
        for t in captured:
            t.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager[0], captured))


def test_large_tables_captured_and_with_every_slot_taken():
    """Tables beyond the launches' arguments: from page-locked memory, by value under capture, and by value when
    other threads hold every slot of page-locked memory."""
    from accdfl_amd.core import norms, wsum

    sizes = [1 + i * 53 % 3000 for i in range(60)]
    center, models, weights = _round(40, sizes, "bf16", seed=22)
    outs = [torch.zeros_like(c) for c in center]
    want, wn, added = no.bounded(models, weights, center, 0.5)

    def check(norms_got):
        torch.cuda.synchronize()
        no.assert_norm(norms_got, wn, sum(sizes))
        for o, w, a in zip(outs, want, added):
            no.assert_close(o, w, sum(sizes), a)
            o.zero_()

    run = lambda: norms.wsum_bounded_multi(models, weights, center, 0.5, outs)  # noqa: E731
    for _ in range(20):  # more calls than slots
        got = run()
    check(got)
    ring = wsum.table_ring(torch.device("cuda", 0))
    taken = [ring.take(8) for _ in range(ring.SLOTS)]
    assert ring.take(8, wait=False) is None
    check(run())
    for idx, _, _ in taken:
        ring.done(idx, torch.cuda.current_stream())
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        check(run())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        captured = run()
    for _ in range(3):
        run()
        for o in outs:
            o.zero_()
        captured.zero_()
        torch.cuda.synchronize()
        g.replay()
        check(captured)


def test_released_storages_are_refused():
    from accdfl_amd.core import norms

    kept, freed = torch.ones(64, device="cuda"), torch.ones(64, device="cuda")
    part = freed[16:32]
    freed.untyped_storage().resize_(0)
    for bad in (freed, part):
        with pytest.raises(ValueError, match="outside its storage"):
            norms.global_norm([kept, bad])
        with pytest.raises(ValueError, match="outside its storage"):
            norms.clip_global_norm_([kept, bad], 1.0)
        with pytest.raises(ValueError, match="outside its storage"):
            norms.update_norms([[bad]], [torch.zeros(bad.shape, device="cuda")])
        with pytest.raises(ValueError, match="outside its storage"):
            norms.wsum_bounded([torch.zeros(bad.shape, device="cuda")], [1.0], bad, 1.0)
    assert norms.global_norm([kept]).item() == 8.0


def test_error_if_nonfinite_is_refused_under_capture():
    from accdfl_amd.core.norms import clip_global_norm_

    t = _rand(100)
    clip_global_norm_([t], 1.0)
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        u = t * 2
        with pytest.raises(RuntimeError, match="captured"):
            clip_global_norm_([u], 1.0, error_if_nonfinite=True)
    torch.cuda.synchronize()


def test_results_do_not_depend_on_the_run():
    from accdfl_amd.core.norms import global_norm, wsum_bounded

    t = _rand(3_000_001, "f32", 0.5, 15)
    first = global_norm([t], 1.0)
    (center,), models, weights = _round(7, [500_001], "bf16", seed=16)
    peers = [m[0] for m in models]
    out, norms = wsum_bounded(peers, weights, center, 5.0)
    for _ in range(10):
        assert torch.equal(global_norm([t], 1.0), first)
        o, n = wsum_bounded(peers, weights, center, 5.0)
        assert torch.equal(o, out) and torch.equal(n, norms)


def test_offsets_beyond_32_bits():
    """A tensor of more than 2^32 bytes and 2^31 elements: its last element counts and is written."""
    from accdfl_amd.core.norms import clip_global_norm_, global_norm, wsum_bounded

    n = (1 << 31) + 4099
    t = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    t[0], t[(1 << 31) + 1], t[n - 1] = 3.0, 4.0, 12.0
    assert float(global_norm([t])) == 13.0
    # 13 / 2 + the norm's eps: the products are 1.5, 2 and 6 within a step of bf16
    assert float(clip_global_norm_([t], 6.5)) == 13.0
    assert [float(t[i]) for i in (0, (1 << 31) + 1, n - 1)] == [1.5, 2.0, 6.0] and float(t[5]) == 0.0
    center = torch.zeros_like(t)
    out, norms = wsum_bounded([t], [1.0], center, 3.25, out=center)
    assert float(norms[0]) == 6.5
    assert [float(out[i]) for i in (0, (1 << 31) + 1, n - 1)] == [0.75, 1.0, 3.0] and float(out[5]) == 0.0


def test_sharded_bounded_with_the_kernels():
    import test_norms

    test_norms.run_sharded(2, 5, 4001, hip=True)


def test_without_the_walk_extension(monkeypatch):
    """The tables made in Python give the same bits."""
    from accdfl_amd import _lib
    from accdfl_amd.core import norms
    from accdfl_amd.core.gradient_aggregation.norm_bounded import NormBoundedFedAvg

    center, models, weights = _round(4, [100, 0, 5001], "bf16", seed=17)
    outs, outs2 = [torch.zeros_like(c) for c in center], [torch.zeros_like(c) for c in center]
    a = norms.wsum_bounded_multi(models, weights, center, 1.0, outs)
    clipped, n = norms.clip_global_norm(models[0], 0.5)
    nets, c, w = _net_case("cuda:0")
    mean = NormBoundedFedAvg(3.0, c).aggregate(nets, w)
    monkeypatch.setattr(_lib, "_walk_mod", None)
    monkeypatch.setattr(_lib, "_walk_tried", True)
    version = outs2[0]._version
    b = norms.wsum_bounded_multi(models, weights, center, 1.0, outs2)
    assert outs2[0]._version > version
    clipped2, n2 = norms.clip_global_norm(models[0], 0.5)
    assert torch.equal(a, b) and torch.equal(n, n2)
    for x, y in zip(outs + clipped, outs2 + clipped2):
        assert torch.equal(x, y)
    mean2 = NormBoundedFedAvg(3.0, c).aggregate(nets, w)
    assert all(torch.equal(x, y) for x, y in zip(mean.parameters(), mean2.parameters()))
