"""The norm operators at the ends of their ranges and of their contract: what a 16-bit average does with values and shares
that float32 does not hold, which calls are refused, and what a refused call leaves as it was.  norms_oracle.py states the
definitions and how far a correct result may be off.  Run on the MI355X: -m gpu."""
import copy
import math

import numpy as np
import pytest
import torch
from torch import nn

import norms_oracle as no
from test_gpu_norms import DT, INF, _list, _native, _rand, _round  # noqa: F401 (the fixture is used by being here)

pytestmark = pytest.mark.gpu


def _row(values, dtype="bf16"):
    return torch.tensor(values, dtype=torch.float64).to(DT[dtype]).cuda()


def _assert_average(out, peers, weights, center, bound):
    want, _, added = no.bounded([[p] for p in peers], weights, [center], bound)
    no.assert_close(out, want[0], center.numel() + len(peers), added[0])


# ------------------------------------------------------------------------- averages of 16-bit types in 64 bits
# No term of these cases, or none before it is divided, lies in float32's normal range: the definition in 64 bits does.
@pytest.mark.parametrize("peers, weights, center, bound", [
    ([3e38], [1.0], -3e38, INF),
    ([3e38, 3e38], [0.5, 0.5], -3e38, INF),
    ([-3e38], [0.9], 1e38, INF),
    ([3e38] * 130, [1.0 / 130] * 130, -3e38, INF),
    ([3e38, 3e38, 3e38], [3.0, -2.5, 0.25], 0.0, INF),
    ([1.0, 1.0, 1.0], [3e38, 3e38, -6e38], 0.0, INF),
    ([1.0, 2.0], [1e-42, 3e-44], 0.0, INF),
    ([3e38, 1.0], [1e-42, 1e-43], 1e-5, INF),
    ([3e38, 0.5, 0.25], [1e-39, 0.25, 0.25], 0.0, INF),
    ([1e20, -1e20], [1e30, 1e30], 0.0, INF),
], ids=str)
def test_bf16_averages_beyond_float32(peers, weights, center, bound):
    from accdfl_amd.core.norms import wsum_bounded

    for numel in (1, 7, 512, 1500):
        c = torch.full((numel,), center, dtype=torch.bfloat16, device="cuda")
        ps = [torch.full_like(c, p) for p in peers]
        out, _ = wsum_bounded(ps, weights, c, bound)
        _assert_average(out, ps, weights, c, bound)


@pytest.mark.parametrize("weights", [[6e38, 6e38, -1.2e39], [1e-44, 1e-42, 0.0], [3e-45, 0.5, 0.25], [1e60, -1e60, 1.0]], ids=str)
def test_f16_averages_with_weights_beyond_float32(weights):
    from accdfl_amd.core.norms import wsum_bounded

    large = max(abs(w) for w in weights) > 1
    # powers of two: every product and sum of the definition is exact in 64 bits, so the large terms cancel to nothing
    c = torch.zeros(1000, dtype=torch.float16, device="cuda")
    ps = [torch.full_like(c, 0.125) for _ in weights]
    out, _ = wsum_bounded(ps, weights, c, INF)
    exact = torch.full((1000,), 0.125 * (1.0 if weights[0] == 1e60 else 0.0) if large else 0.125 * sum(weights), dtype=torch.float64)
    no.assert_close(out, exact, 1000)
    c = _rand(3001, "f16", 0.5, 1)
    ps = [_rand(3001, "f16", 0.5, 2 + k) for k in range(len(weights))]
    if large:
        ps = [ps[0].clone() for _ in ps]
    out, _ = wsum_bounded(ps, weights, c, INF)
    if large:
        # The terms cancel, but the rounding of products of 1e38 |d| and more to 64 bits, 2^-53 of them, is 1e22 |d|: any
        # result of float16, infinities too, is within what 64 bits allow wherever |d| > 1e-15; d = 0 is exact.
        d = ps[0].double() - c.double()
        assert float(d[d != 0].abs().min()) > 1e-15
        assert not bool(torch.isnan(out).any()) and torch.equal(out[d == 0], c[d == 0])
    else:
        _assert_average(out, ps, weights, c, INF)


@pytest.mark.parametrize("n", [1, 2, 9, 128])
@pytest.mark.parametrize("bound", [1.0, 1e-3, 1e-4, 1e-5, 1e-30])
def test_an_outlier_of_any_size_is_bounded(bound, n):
    """One peer of norm 3e38 and more moves the average by its weight times the bound, however small that is: its share,
    near 1e-45 and below, is no normal float32."""
    from accdfl_amd.core.norms import wsum_bounded

    c = torch.zeros(2000, dtype=torch.bfloat16, device="cuda")
    far = _rand(2000, "f64", 1e37, 3).to(torch.bfloat16)
    far[777] = 3e38
    peers = [far] + [c.clone() for _ in range(n - 1)]
    out, _ = wsum_bounded(peers, [1.0 / 128] * n, c, bound)
    # one term, no sum: within half a step of the definition
    want = far.double().cpu() * (bound / no.norm([far]) / 128)
    no.assert_close(out, want, 2000 + n)
    assert abs(no.norm([out]) * 128 - bound) <= 2.0 ** -8 * bound


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n", [2, 5, 8, 11, 70])
def test_an_outlier_beside_ordinary_peers(n, dtype):
    """The round that holds a peer beyond float32 and the others alike are off by no more than any other round."""
    from accdfl_amd.core.norms import wsum_bounded, wsum_bounded_multi

    sizes = [5, 1025, 6007]
    center, models, weights = _round(n, sizes, dtype, seed=21)
    for t in models[n // 2]:
        t.copy_(_rand(t.shape, "f64", 1.0, 22).to(DT[dtype]) * (3e37 if dtype == "bf16" else 6e3))
    outs = [torch.empty_like(c) for c in center]
    got = wsum_bounded_multi(models, weights, center, 0.5, outs)
    want, wn, added = no.bounded(models, weights, center, 0.5)
    # a norm is returned in float32 (beyond its largest value: infinite) and judged in 64 bits
    no.assert_norm(got, [w if w <= torch.finfo(torch.float32).max else INF for w in wn], sum(sizes))
    for o, w, a in zip(outs, want, added):
        no.assert_close(o, w, sum(sizes) + n, a)
    out, _ = wsum_bounded([m[2] for m in models], weights, center[2], 0.5, out=center[2].clone())
    _assert_average(out, [m[2] for m in models], weights, center[2], 0.5)


@pytest.mark.parametrize("own", [False, True])
def test_a_slab_with_an_outlier(own):
    from accdfl_amd.core.peer_slab import PeerSlab

    total, n = 30_011, 6
    center = _rand(total, "bf16", 0.5, 31)
    peers = [(center.double() + _rand(total, "f64", 0.1, 40 + k)).to(torch.bfloat16) for k in range(n)]
    peers[2] = torch.full_like(center, -3e38)
    slab = PeerSlab([(total,)], torch.bfloat16, capacity=n)
    for p in peers:
        slab.stage_flat(p)
    around = center if own else peers[0]
    weights = [1.0 / n] * n
    for bound in (2.0, 1e-6, INF):
        out, _ = slab.reduce_bounded(bound, weights, center=center if own else None)
        _assert_average(out[:total], peers, weights, around, bound)


@pytest.mark.parametrize("n", [1, 2, 9])
def test_given_norms_below_the_updates_own(n):
    """sq_norms are taken as they are: float32's range, which they seem to promise, is passed all the same."""
    from accdfl_amd.core.norms import wsum_bounded

    c = torch.full((1500,), -3e38, dtype=torch.bfloat16, device="cuda")
    peers = [torch.full_like(c, 3e38) for _ in range(n)]
    sq = torch.ones(n, dtype=torch.float64, device="cuda")
    for weight in (0.25, 1.0):
        out, norms = wsum_bounded(peers, [weight / n] * n, c, 2.0, sq_norms=sq)
        want, _, added = no.bounded([[p] for p in peers], [weight / n] * n, [c], 2.0, norms=[1.0] * n)
        no.assert_close(out, want[0], 1500 + n, added[0])
        assert bool((norms == 1.0).all())


def test_squared_norms_are_read_from_what_their_storage_holds():
    from accdfl_amd.core.norms import wsum_bounded

    c, sq = _rand(100), torch.ones(2, dtype=torch.float64, device="cuda")
    freed = sq.clone()
    freed.untyped_storage().resize_(0)
    for bad in (freed, torch._neg_view(sq), sq[:1].expand(2), sq.float()):
        with pytest.raises(ValueError, match="sq_norms"):
            wsum_bounded([c, c], [0.5, 0.5], c, 1.0, sq_norms=bad)


# ------------------------------------------------------------------------------------------ overlapping outputs
def _overlapping():
    """(name, the tensors to write): each list has an element that is written twice."""
    buf = torch.arange(120, dtype=torch.float32, device="cuda")
    m = buf.view(10, 12)
    gapped = m[:, :3]
    return [
        ("the same view twice", [gapped, gapped]),
        ("columns that cross", [m[:, :3], m[:, 2:5]]),
        ("steps of two and four", [buf[::2], buf[::4]]),
        ("a column of a whole", [m, m[:, 3:4]]),
        ("dense beside gapped", [buf[:24], m[:, 11]]),
        ("windows", [buf.as_strided((3, 3), (1, 1))]),
        ("a window that meets itself late", [buf.as_strided((5, 4), (3, 4))]),
        ("rows and their transpose", [m[:5, :5], m[:5, :5].t()]),
    ]


def test_overlapping_outputs_with_gaps_are_refused():
    from accdfl_amd import _lib
    from accdfl_amd.core.norms import clip_global_norm, clip_global_norm_, wsum_bounded_multi

    for name, outs in _overlapping():
        base = outs[0]._base if outs[0]._base is not None else outs[0]
        before = base.clone()
        versions = [o._version for o in outs]
        fresh = [torch.ones(o.shape, device="cuda") for o in outs]
        for call in (lambda: clip_global_norm_(outs, 0.1), lambda: clip_global_norm(fresh, 0.1, outs=outs),
                     lambda: wsum_bounded_multi([fresh], [0.5], fresh, 1.0, outs),
                     lambda: wsum_bounded_multi([outs], [0.5], outs, 1.0, outs)):
            with pytest.raises((ValueError, _lib.DlaggError), match="overlap|share memory"):
                call()
            assert torch.equal(base, before), name
        assert [o._version for o in outs] == versions, name


def test_outputs_that_cross_other_inputs_are_refused():
    from accdfl_amd import _lib
    from accdfl_amd.core.norms import clip_global_norm, wsum_bounded_multi

    m = _rand((10, 12), "f32", 1.0, 3)
    fresh = torch.ones(10, 3, device="cuda")
    for tensors, outs in (([m[:, :3]], [m[:, 1:4]]), ([m[:, :3], m[:, 3:6]], [m[:, 3:6], fresh]),
                          ([m[:5, :5]], [m[:5, :5].t()]), ([m[:3, :3].expand(3, 3)], [m[:6:2, :3]])):
        before = m.clone()
        with pytest.raises(_lib.DlaggError, match="overlap"):
            clip_global_norm(tensors, 0.1, outs=outs)
        with pytest.raises(_lib.DlaggError, match="overlap"):
            wsum_bounded_multi([tensors], [1.0], tensors, 0.1, outs)
        assert torch.equal(m, before)


def test_interleaved_views_of_one_base_are_not_refused():
    """Views with gaps that share no element: columns, rows, every other element, and one that lies in another's gaps."""
    from accdfl_amd.core.norms import clip_global_norm_, wsum_bounded_multi

    def views(m):
        crossed = m.as_strided((2, 2), (3, 2), m.storage_offset() + 9 * 12 + 6)  # columns 6, 8, 9 and 11 of row 9
        return [m[:, 0], m[:, 1:4], m[::2, 4:6], m[1::2, 4:6], m.view(-1)[7::12], m[3:4, 8:10], crossed]

    m = _rand((12, 12), "f32", 1.0, 5)
    rest = torch.ones_like(m, dtype=torch.bool)
    for v in views(rest):
        v.zero_()
    kept = m.clone()
    want, _ = no.clip(views(m), 0.2)
    clip_global_norm_(views(m), 0.2)
    for v, w in zip(views(m), want):
        no.assert_close(v, w, 144)
    assert torch.equal(m[rest], kept[rest])
    peer = _rand((12, 12), "f32", 1.0, 6)
    want, wn, added = no.bounded([views(peer)], [0.5], views(m), 0.3)
    wsum_bounded_multi([views(peer)], [0.5], views(m), 0.3, views(m))
    for v, w, a in zip(views(m), want, added):
        no.assert_close(v, w, 144, a)
    assert torch.equal(m[rest], kept[rest])


# ------------------------------------------------------------------------------- what a refused clip leaves alone
def _bits(t):
    return t.view({2: torch.int16, 4: torch.int32, 8: torch.int64}[t.element_size()]).clone()


@pytest.mark.parametrize("p", [2.0, 1.0, INF])
@pytest.mark.parametrize("bad", [math.nan, INF, -INF])
def test_a_clip_refused_for_its_norm_writes_nothing(bad, p):
    from accdfl_amd.core.norms import clip_global_norm, clip_global_norm_

    for dtype in DT:
        base = _rand((50, 40), dtype, 1.0, 2)
        ts = [_rand(9, dtype), _rand(70_001, dtype, 1.0, 1), base[:, 3:20]]  # the last is written through a copy
        ts[1][33_333] = bad
        sent = [torch.full_like(t, 7.0) for t in ts]
        before, versions = [_bits(t) for t in ts + sent], [t._version for t in ts + sent]
        with pytest.raises(RuntimeError, match="not finite"):
            clip_global_norm_(ts, 1.0, p, error_if_nonfinite=True)
        with pytest.raises(RuntimeError, match="not finite"):
            clip_global_norm(ts, 1.0, p, error_if_nonfinite=True, outs=sent)
        assert all(torch.equal(_bits(t), b) for t, b in zip(ts + sent, before))
        assert [t._version for t in ts + sent] == versions
        ts[1][33_333] = 0.0
        versions = [t._version for t in ts]
        want, wn = no.clip(ts, 1.0, p)
        no.assert_norm(clip_global_norm_(ts, 1.0, p, error_if_nonfinite=True), wn, 80_000)
        for t, w in zip(ts, want):
            no.assert_close(t, w, 80_000)
        assert all(t._version > v for t, v in zip(ts, versions))


def test_a_refused_call_moves_no_version():
    from accdfl_amd import _lib
    from accdfl_amd.core.norms import clip_global_norm_, wsum_bounded

    t = _rand(100)
    views = [t[:60], t[50:]]
    with pytest.raises(_lib.DlaggError, match="overlap"):
        clip_global_norm_(views, 0.1)
    with pytest.raises(_lib.DlaggError, match="overlap"):
        wsum_bounded([t[:50]], [1.0], t[:50], 1.0, out=t[1:51])
    assert t._version == 0


def test_without_the_walk_extension_a_refused_call_moves_no_version(monkeypatch):
    from accdfl_amd import _lib

    monkeypatch.setattr(_lib, "walk_module", lambda: None)
    test_a_refused_call_moves_no_version()
    test_a_clip_refused_for_its_norm_writes_nothing(math.nan, 2.0)


# ---------------------------------------------------------------------------------------- what is written has moved on
@pytest.mark.parametrize("dtype", list(DT))
def test_a_slab_s_output_has_moved_on(dtype):
    from accdfl_amd.core.peer_slab import PeerSlab

    slab = PeerSlab([(5003,)], DT[dtype], capacity=3)
    for k in range(3):
        slab.stage_flat(_rand(5003, dtype, 1.0, k))
    out = torch.zeros(5003, dtype=DT[dtype], device="cuda")
    version = out._version
    assert slab.reduce_bounded(0.5, out=out)[0] is out and out._version > version
    w = torch.ones(5003, dtype=DT[dtype], device="cuda", requires_grad=True)
    loss = (w * out).sum()
    slab.reduce_bounded(0.25, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("layout", ["tiled", "rows"])
def test_a_slab_s_tensors_are_what_their_storages_hold(layout):
    from accdfl_amd.core.peer_slab import PeerSlab

    slab = PeerSlab([(40, 50), (3,)], torch.float32, capacity=2, layout=layout)
    peers = [_rand(2003, "f32", 1.0, k) for k in range(2)]
    for p in peers:
        slab.stage_flat(p)
    freed = torch.ones(2003, device="cuda")
    part, whole = freed[:2000].view(40, 50), torch.ones(3, device="cuda")
    freed.untyped_storage().resize_(0)
    for kw in (dict(out=freed), dict(center=freed), dict(center=[part, whole])):
        with pytest.raises(ValueError, match="storage"):
            slab.reduce_bounded(1.0, **kw)
    # a negated view is read, and where it can be written, as what it stands for
    center, out = _rand(2003, "f32", 1.0, 9), torch.zeros(2003, device="cuda")
    if layout == "tiled":
        with pytest.raises(ValueError, match="negated"):
            slab.reduce_bounded(1.0, out=torch._neg_view(out))
    else:
        slab.reduce_bounded(1.0, [0.5, 0.5], center=center, out=torch._neg_view(out))
        _assert_average(-out, peers, [0.5, 0.5], center, 1.0)
    out, _ = slab.reduce_bounded(1.0, [0.5, 0.5], center=torch._neg_view(center))
    _assert_average(out, peers, [0.5, 0.5], -center, 1.0)


# ------------------------------------------------------------------------------------------------------- 64 GiB
def test_an_average_of_64_gib_and_more():
    """One more unit than a launch has workgroups for: the first ones walk.  In place, around the output."""
    from accdfl_amd.core.norms import wsum_bounded

    n = 2 ** 26 * 512 + 517
    if torch.cuda.mem_get_info()[0] < 2 * 2 * n + (8 << 30):
        pytest.skip("needs 136 GiB of free memory")
    center = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    peer = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    at = [0, 1, 511, 512, 513, 1023, 1024, 1500, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, n // 2, n - 518, n - 6, n - 5, n - 1]
    for i, a in enumerate(at):
        peer[a] = float(i + 1)
        center[a] = 1.0
    out, norms = wsum_bounded([peer], [0.5], center, INF, out=center)
    got = [float(out[a]) for a in at]
    rest = [float(out[a + 2].abs()) for a in at if a + 2 < n and a + 2 not in at]
    no.assert_norm(norms, [math.sqrt(sum(i * i for i in range(len(at))))], 1000)
    del center, peer, out
    torch.cuda.empty_cache()
    assert got == [1.0 + 0.5 * i for i in range(len(at))]
    assert not any(rest)


# ------------------------------------------------------------------------------------------------ CPU rounds at once
class _Nested(nn.Module):
    """Averages other models while it is being copied."""

    def __init__(self, seed, others=()):
        super().__init__()
        self.w = nn.Parameter(_rand((300, 40), "f32", 0.1, seed).cpu())
        self.others, self.made = others, []

    def __deepcopy__(self, memo):
        twin = _Nested.__new__(_Nested)
        memo[id(self)] = twin
        nn.Module.__init__(twin)
        twin.others, twin.made = (), []
        twin.w = copy.deepcopy(self.w, memo)
        if self.others:
            from accdfl_amd.core.gradient_aggregation.norm_bounded import NormBoundedFedAvg

            self.made.append(NormBoundedFedAvg(1.0).aggregate(list(self.others), None))
        return twin


def test_a_cpu_round_within_a_cpu_round():
    from accdfl_amd.core.gradient_aggregation.norm_bounded import NormBoundedFedAvg, release_staging

    others = [_Nested(50 + k) for k in range(3)]
    models = [_Nested(60, others)] + [_Nested(61 + k) for k in range(2)]
    out = NormBoundedFedAvg(2.0).aggregate(models, [0.5, 0.25, 0.25])
    (inner,) = models[0].made
    for got, ms, weights, bound in ((out, models, [0.5, 0.25, 0.25], 2.0), (inner, others, [1 / 3] * 3, 1.0)):
        want, _, added = no.bounded([[m.w] for m in ms], weights, [ms[0].w], bound)
        no.assert_close(got.w, want[0], 12_000, added[0])
    release_staging()


# --------------------------------------------------------------------------- how exact, and the largest forms in full
@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("n", [1, 2, 9, 16, 130])
def test_averages_in_64_bits_are_off_by_one_rounding_a_step(n, dtype):
    """Without a bound the shares are the weights.  In 64 bits the difference, the product with its addition, and the
    centre's addition round once each: N + 3 times 2^-53 of M = |c| + sum_k |w_k d_k| at most, and then the result by half a
    step.  The reference is carried in 80 bits, which adds (N + 3) 2^-64 M."""
    from accdfl_amd.core.norms import wsum_bounded

    (center,), models, weights = _round(n, [20_011], dtype, seed=50, scale=0.5)
    out, _ = wsum_bounded([m[0] for m in models], weights, center, INF)
    c = center.cpu().numpy().astype(np.longdouble)
    want, mag = c.copy(), np.abs(c)
    for (m,), w in zip(models, weights):
        d = np.longdouble(w) * (m.cpu().numpy().astype(np.longdouble) - c)
        want, mag = want + d, mag + np.abs(d)
    off = np.abs(out.cpu().numpy().astype(np.longdouble) - want)
    half = torch.finfo(DT[dtype]).eps / 2
    assert bool((off <= half * np.abs(want) + (n + 3) * (2.0 ** -53 + 2.0 ** -64) * (1 + half) * mag).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "f64"])
@pytest.mark.parametrize("in_place", [False, True])
def test_a_clip_beyond_the_infinity_cache_in_full(dtype, in_place):
    """Over 256 MB a clip streams past the caches: every element, in place and out of place, tensors at odd starts."""
    from accdfl_amd.core.norms import clip_global_norm

    sizes = [300 * (1 << 20) // DT[dtype].itemsize, 5, 1_000_003]
    buf = torch.randn(sum(sizes), device="cuda", generator=torch.Generator("cuda").manual_seed(3)).mul_(0.01).to(DT[dtype])
    ts = list(torch.split(buf, sizes[::-1]))
    kept = buf.clone()
    sent = buf if in_place else torch.full_like(buf, 7.0)
    outs, norm = clip_global_norm(ts, 0.5, outs=list(torch.split(sent, sizes[::-1])))
    exact = math.sqrt(sum(float(k.double().square().sum()) for k in torch.split(kept, 1 << 24)))
    no.assert_norm(norm, exact, buf.numel())
    ratio = 0.5 / (exact + no.CLIP_EPS)
    # the norm, of up to 1.6e8 terms on either side, is off by 2^-53 of the longest chain of sums: below 2^-30 by far
    half = torch.finfo(DT[dtype]).eps / 2 + (0.0 if dtype == "f64" else 2.0 ** -24) + 2.0 ** -30
    least = torch.finfo(DT[dtype]).smallest_normal * torch.finfo(DT[dtype]).eps / 2
    for s, k in zip(torch.split(sent, 1 << 24), torch.split(kept, 1 << 24)):
        want = k.double() * ratio
        assert bool(((s.double() - want).abs() <= half * want.abs() + least).all())
    if not in_place:
        assert torch.equal(buf, kept)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "f64"])
def test_an_average_beyond_the_infinity_cache_in_full(dtype):
    """Rounds of 8 peers and more over 256 MB run fewer waves at once: every element."""
    from accdfl_amd.core.norms import wsum_bounded_multi

    n, sizes = 9, [2_700_001 * 4 // DT[dtype].itemsize * 3, 11, 70_001]
    gen = torch.Generator("cuda").manual_seed(4)
    make = lambda scale: [torch.randn(s, device="cuda", generator=gen).mul_(scale).to(DT[dtype]) for s in sizes]  # noqa: E731
    center = make(0.5)
    models = [[(c + d).to(DT[dtype]) for c, d in zip(center, make(0.01 * (1 + k % 3)))] for k in range(n)]
    assert sum(sizes) * DT[dtype].itemsize * (n + 1) > 256 << 20
    weights = [(k + 1) / 45 for k in range(n)]
    bound = 0.015 * math.sqrt(sum(sizes))
    outs = [torch.empty_like(c) for c in center]
    norms = wsum_bounded_multi(models, weights, center, bound, outs)
    exact = [math.sqrt(sum(float((m.double() - c.double()).square().sum()) for m, c in zip(ms, center))) for ms in models]
    no.assert_norm(norms, exact, sum(sizes))
    assert min(exact) < bound < max(exact)
    info = torch.finfo(DT[dtype])
    steps = 2.0 ** -30 + (2.0 ** -24 * (n + 3) if DT[dtype].itemsize == 2 else 0.0)  # the norms' own error; 32-bit sums
    for i, o in enumerate(outs):
        c = center[i].double()
        want, mag = c.clone(), c.abs()
        for ms, a in zip(models, no.shares(exact, weights, bound)):
            d = a * (ms[i].double() - c)
            want, mag = want + d, mag + d.abs()
        half = info.eps / 2 + (0.0 if dtype == "f64" else 2.0 ** -24)
        assert bool(((o.double() - want).abs() <= half * want.abs() + steps * mag + info.smallest_normal * info.eps / 2).all())
