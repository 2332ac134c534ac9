"""Norms over many tensors, clipping by them and norm-bounded averages: what needs no GPU — refusals of the C ABI and
of the Python calls, the aggregator's dispatch, and the bucket-sharded form over gloo ranks with the 64-bit
definitions in the kernels' place."""
import ctypes
import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp
from torch import nn

import norms_oracle as no
from test_sharding_gloo import _free_port

VP = ctypes.c_void_p


@pytest.fixture(scope="module")
def L():
    from accdfl_amd import _lib

    _lib.build()
    return _lib.lib()


def _err(L, rc):
    return rc, L.so.dla_last_error().decode()


def _ints(*v):
    return (ctypes.c_int * len(v))(*v)


def _longs(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _ptrs(*v):
    return (VP * len(v))(*v)


# None of these reaches a launch: every call below fails its checks first.
A, B, WS, BIG = 0x10000, 0x20000, 0x900000, 1 << 30


def _norm(L, n=1, codes=None, ptrs=None, numels=None, norm=2, out_code=0, out=0x40000, counter=None, ws=WS, nbytes=BIG):
    return _err(L, L.so.dla_norm(n, codes or _ints(0), ptrs or _ptrs(A), numels or _longs(4), norm, out_code, out, counter,
                                 ws, nbytes, None))


@pytest.mark.parametrize("kw, text", [
    (dict(n=-1), "n_tensors < 0"),
    (dict(codes=_ints(7)), "unknown dtype"),
    (dict(numels=_longs(-1)), "bad element count"),
    (dict(numels=_longs(1 << 60)), "bad element count"),
    (dict(ptrs=_ptrs(None)), "null"),
    (dict(ptrs=_ptrs(A + 2)), "not aligned"),
    (dict(codes=_ints(1), ptrs=_ptrs(A + 1)), "not aligned"),
    (dict(norm=3), "unknown norm"),
    (dict(out_code=1), "F32 or F64"),
    (dict(out_code=3, out=0x40004), "F32 or F64"),
    (dict(out=None), "null out"),
    (dict(counter=0x50002), "counter"),
    (dict(ws=None), "workspace"),
    (dict(ws=WS + 4), "workspace"),
    (dict(nbytes=64), "workspace"),
])
def test_norm_refusals(L, kw, text):
    rc, msg = _norm(L, **kw)
    assert rc == -1 and text in msg, (rc, msg)


def _clip(L, n=1, codes=None, ptrs=None, outs=None, numels=None, max_norm=1.0, eps=1e-6, norm_out=None, counter=None,
          ws=WS, nbytes=BIG):
    return _err(L, L.so.dla_norm_clip(n, codes or _ints(0), ptrs or _ptrs(A), outs or _ptrs(B), numels or _longs(4), 2,
                                      max_norm, eps, 0, norm_out, counter, ws, nbytes, None))


@pytest.mark.parametrize("kw, rc_want, text", [
    (dict(max_norm=-1.0), -1, "max_norm"),
    (dict(max_norm=math.nan), -1, "max_norm"),
    (dict(eps=-1.0), -1, "eps"),
    (dict(eps=0.0), -1, "eps"),
    (dict(outs=_ptrs(None)), -1, "null"),
    (dict(outs=_ptrs(B + 1)), -1, "not aligned"),
    (dict(norm_out=0x40002), -1, "F32 or F64"),
    (dict(counter=0x50001), -1, "counter"),
    (dict(ws=None), -1, "workspace"),
    # an output a part of its own input, of another input, of another output; the same tensor twice
    (dict(outs=_ptrs(A + 4)), -2, "overlaps"),
    (dict(n=2, codes=_ints(0, 0), ptrs=_ptrs(A, B), outs=_ptrs(B, 0x30000), numels=_longs(4, 4)), -2, "overlaps"),
    (dict(n=2, codes=_ints(0, 0), ptrs=_ptrs(A, B), outs=_ptrs(0x30000, 0x30008), numels=_longs(4, 4)), -2, "overlap"),
    (dict(n=2, codes=_ints(0, 0), ptrs=_ptrs(A, A), outs=_ptrs(A, A), numels=_longs(4, 4)), -2, "overlap"),
    (dict(n=2, codes=_ints(0, 0), ptrs=_ptrs(A, A + 8), outs=_ptrs(A, A + 8), numels=_longs(4, 4)), -2, "overlap"),
])
def test_norm_clip_refusals(L, kw, rc_want, text):
    rc, msg = _clip(L, **kw)
    assert rc == rc_want and text in msg, (rc, msg)


def _bounded(L, n=1, peers=2, codes=None, ptrs=None, centers=None, outs=None, numels=None, weights=True, max_norm=1.0,
             norms=None, counters=None, ws=WS, nbytes=BIG, sq=None):
    return _err(L, L.so.dla_wsum_bounded(
        n, codes or _ints(0), ptrs or _ptrs(A, B), centers or _ptrs(0x30000), outs or _ptrs(0x40000), numels or _longs(4),
        (ctypes.c_double * max(1, peers))(*[0.5] * max(1, peers)) if weights else None, peers, max_norm,
        ctypes.cast(sq, ctypes.POINTER(ctypes.c_double)) if sq else None, 0, norms, counters,
        None, 0, ws, nbytes, None))


@pytest.mark.parametrize("kw, rc_want, text", [
    (dict(peers=0), -1, "n_peers"),
    (dict(peers=2049), -1, "n_peers"),
    (dict(n=-1), -1, "n_tensors"),
    (dict(codes=_ints(4)), -1, "unknown dtype"),
    (dict(numels=_longs(-3)), -1, "bad element count"),
    (dict(centers=_ptrs(None)), -1, "centre tensor 0"),
    (dict(ptrs=_ptrs(A, None)), -1, "peer 1"),
    (dict(ptrs=_ptrs(A, B + 2)), -1, "peer 1"),
    (dict(outs=_ptrs(None)), -1, "out 0"),
    (dict(weights=False), -1, "weights"),
    (dict(max_norm=-0.5), -1, "max_norm"),
    (dict(max_norm=math.nan), -1, "max_norm"),
    (dict(norms=0x50002), -1, "norms"),
    (dict(counters=0x50002), -1, "counters"),
    (dict(sq=0x50004), -1, "squared norms"),
    (dict(ws=None), -1, "workspace"),
    (dict(nbytes=128), -1, "workspace"),
    (dict(outs=_ptrs(B + 4)), -2, "peer 1"),
    (dict(outs=_ptrs(0x30000 - 8)), -2, "centre"),
    (dict(n=2, codes=_ints(0, 0), ptrs=_ptrs(A, B, A + 64, B + 64), centers=_ptrs(0x30000, 0x30040),
          outs=_ptrs(0x30040, 0x50000), numels=_longs(4, 4)), -2, "centre tensor 1"),
    (dict(n=2, codes=_ints(0, 0), ptrs=_ptrs(A, B, A + 64, B + 64), centers=_ptrs(0x30000, 0x30040),
          outs=_ptrs(0x50000, 0x50004), numels=_longs(4, 4)), -2, "outputs overlap"),
])
def test_bounded_refusals(L, kw, rc_want, text):
    rc, msg = _bounded(L, **kw)
    assert rc == rc_want and text in msg, (rc, msg)


@pytest.mark.parametrize("kw, rc_want, text", [
    (dict(dtype=9), -1, "unknown dtype"),
    (dict(tile=6), -1, "power of two"),
    (dict(tile=2), -1, "power of two"),
    (dict(base=None), -1, "base"),
    (dict(base=A + 8), -1, "16-byte"),
    (dict(rows=1), -1, "slab_rows"),
    (dict(rows=1 << 60), -1, "beyond any device"),
    (dict(tile=0), -1, "power of two"),
    (dict(tile=1 << 40), -1, "power of two"),
    (dict(n=0), -1, "n_peers"),
    (dict(numel=-1), -1, "element count"),
    (dict(out=None), -1, "null out"),
    (dict(out=0x40002), -1, "aligned"),
    (dict(out=A + 16), -2, "overlaps"),
    (dict(center=0x40010), -2, "overlaps"),
    (dict(max_norm=math.nan), -1, "max_norm"),
])
def test_bounded_slab_refusals(L, kw, rc_want, text):
    a = dict(dtype=0, base=A, tile=8, rows=2, center=None, n=2, numel=20, out=0x40000, max_norm=1.0)
    a.update(kw)
    rc = L.so.dla_wsum_bounded_slab_tiled(a["dtype"], a["base"], a["tile"], a["rows"], a["center"],
                                          (ctypes.c_double * 2)(0.5, 0.5), a["n"], a["numel"], a["max_norm"], a["out"], 0,
                                          None, None, WS, BIG, None)
    rc, msg = _err(L, rc)
    assert rc == rc_want and text in msg, (rc, msg)


def test_workspaces(L):
    assert L.so.dla_norm_workspace(-1) == 0 and L.so.dla_norm_workspace(0) >= 8
    assert L.so.dla_peer_workspace(3, 0) == 0 and L.so.dla_peer_workspace(3, 2049) == 0 and L.so.dla_peer_workspace(-1, 1) == 0
    assert L.so.dla_peer_workspace(110, 128) >= 8 * 110 * 128
    sizes = [L.so.dla_norm_workspace(t) for t in (1, 190, 191, 10_000)]
    assert sizes == sorted(sizes)


def test_python_refusals_that_need_no_device():
    from accdfl_amd.core import norms
    from accdfl_amd.core.gradient_aggregation.norm_bounded import NormBoundedFedAvg

    t = [torch.zeros(3)]
    for bad in (3, 0.5, -1.0, math.nan):
        with pytest.raises(ValueError, match="norm_type"):
            norms.global_norm(t, norm_type=bad)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            norms.clip_global_norm_(t, bad)
        with pytest.raises(ValueError, match="max_norm"):
            norms.wsum_bounded(t, [1.0], t[0], bad)
        with pytest.raises(ValueError, match="max_norm"):
            NormBoundedFedAvg(bad)
    with pytest.raises(IndexError):
        norms.update_norms([], t)
    with pytest.raises(ValueError, match="2049 peers"):
        norms.update_norms([t] * 2049, t)
    with pytest.raises(AssertionError):
        norms.wsum_bounded_multi([t, t], [1.0], t, 1.0, t)
    with pytest.raises(IndexError):
        NormBoundedFedAvg(1.0).aggregate([], None)
    with pytest.raises(AssertionError):
        NormBoundedFedAvg(1.0).aggregate([nn.Linear(2, 2)], [0.5, 0.5])


def test_layout_refusals():
    from accdfl_amd.core.gradient_aggregation.norm_bounded import _check_layout

    a, b = nn.Linear(2, 3), nn.Linear(2, 3)
    assert len(_check_layout([a, b], a)) == 3
    with pytest.raises(RuntimeError, match="model 1 has 1 parameters"):
        _check_layout([a, nn.Linear(2, 3, bias=False)], a)
    with pytest.raises(RuntimeError, match="center is"):
        _check_layout([a, b], nn.Linear(3, 3))
    with pytest.raises(RuntimeError, match="float64"):
        _check_layout([a, nn.Linear(2, 3).double()], a)
    with pytest.raises(TypeError):
        _check_layout([nn.ParameterList([nn.Parameter(torch.zeros(2, dtype=torch.int32), requires_grad=False)])] * 2,
                      nn.ParameterList([nn.Parameter(torch.zeros(2, dtype=torch.int32), requires_grad=False)]))


def test_dense_helpers():
    from accdfl_amd.core.norms import _dense, _same_order

    x = torch.zeros(4, 3, 2)
    assert _dense(x) and _dense(x.transpose(0, 2)) and _dense(x[1]) and _dense(torch.zeros(0, 5)) and _dense(torch.zeros(()))
    assert _dense(torch.zeros(1, 4)[:, :1]) and _dense(torch.zeros(3, 1, 4).expand(3, 1, 4))
    assert not _dense(x[:, :2]) and not _dense(torch.zeros(4, 1).expand(4, 3)) and not _dense(x[..., 0])
    assert not _dense(torch.zeros(8).as_strided((3, 3), (1, 1)))
    for t in (x, x.transpose(0, 2), x[:, :2], x[..., 0], torch.zeros(4, 1).expand(4, 3)):
        assert _dense(t) == torch.ops.aten.is_non_overlapping_and_dense(t)
    assert _same_order(x, torch.ones(4, 3, 2)) and not _same_order(x, torch.zeros(2, 3, 4).transpose(0, 2))


def test_method_is_selected_by_the_settings():
    from accdfl_amd.core.gradient_aggregation import GradientAggregationMethod
    from accdfl_amd.core.gradient_aggregation.fedavg import FedAvg
    from accdfl_amd.core.gradient_aggregation.norm_bounded import NormBoundedFedAvg
    from accdfl_amd.core.model_manager import ModelManager

    assert GradientAggregationMethod.FEDAVG == 1
    model = nn.Linear(2, 2)
    mm = ModelManager(model, SimpleNamespace(gradient_aggregation=GradientAggregationMethod.NORM_BOUNDED_FEDAVG,
                                             max_update_norm=0.25))
    method = mm.get_aggregation_method()
    assert isinstance(method, NormBoundedFedAvg) and method.max_norm == 0.25 and method.center is model
    mm = ModelManager(model, SimpleNamespace(gradient_aggregation=GradientAggregationMethod.FEDAVG))
    assert mm.get_aggregation_method() is FedAvg


def test_the_oracle_sees_a_planted_mistake():
    """The tolerance of the GPU tests is tight enough to tell one wrong share, one skipped element, or a norm that is
    off by a part in 10^6."""
    g = torch.Generator().manual_seed(1)
    c = [torch.randn(1000, generator=g).double()]
    ms = [[c[0] + 0.1 * torch.randn(1000, generator=g).double()] for _ in range(3)]
    want, n, added = no.bounded(ms, [0.3, 0.3, 0.4], c, 1.0)
    no.assert_close(want[0].float(), want[0], 1000, added[0])
    with pytest.raises(AssertionError):
        no.assert_close(no.bounded(ms, [0.3, 0.3, 0.4], c, 1.00001)[0][0].float(), want[0], 1000, added[0])
    bad = want[0].clone()
    bad[999] = c[0][999]
    with pytest.raises(AssertionError):
        no.assert_close(bad.float(), want[0], 1000, added[0])
    with pytest.raises(AssertionError):
        no.assert_norm(torch.tensor(n[0] * (1 + 1e-6), dtype=torch.float32), n[0], 1000)


# ------------------------------------------------------------------------- bucket-sharded, gloo ranks on the CPU
def _oracle_bounded():
    def sq_norms(peers, center):
        return torch.tensor([no.norm([p.double() - center.double()]) ** 2 if p.numel() else 0.0 for p in peers],
                            dtype=torch.float64)

    def average(peers, weights, center, max_norm, sq, out):
        outs, _, _ = no.bounded([[p] for p in peers], weights, [center], max_norm, norms=[math.sqrt(float(s)) for s in sq])
        out.copy_(outs[0])
    return sq_norms, average


def _hip_bounded():
    from accdfl_amd.core import norms

    dev = torch.device("cuda", 0)

    def sq_norms(peers, center):
        return norms.update_norms([[p.to(dev)] for p in peers], [center.to(dev)], squared=True).cpu()

    def average(peers, weights, center, max_norm, sq, out):
        out.copy_(norms.wsum_bounded([p.to(dev) for p in peers], weights, center.to(dev), max_norm,
                                     sq_norms=sq.to(dev))[0].cpu())
    return sq_norms, average


def test_tensors_outside_their_storage_are_seen():
    from accdfl_amd.core.norms import _held

    base = torch.zeros(100)
    views = [base, base[40:60], base[::7], base.view(10, 10).t(), base[3:4].expand(5), base[:0]]
    assert all(_held(v) for v in views)
    base.untyped_storage().resize_(4 * 70)
    assert [_held(v) for v in views] == [False, True, False, False, True, True]
    base.untyped_storage().resize_(0)
    assert [_held(v) for v in views] == [False] * 5 + [True]


def test_sharded_bound_is_checked_before_the_collective():
    from accdfl_amd.core.sharding import BucketShardedFedAvg

    def never(*_):
        raise AssertionError("reached")

    sh = BucketShardedFedAvg(64, torch.float32, device=torch.device("cpu"), bounded=(never, never))
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            sh.reduce_bucket_bounded([torch.zeros(64)], torch.zeros(64), bad)


def _sharded_inputs(n_peers, n_elems):
    g = torch.Generator().manual_seed(n_peers * 1000 + n_elems)
    center = torch.randn(n_elems, generator=g) * 0.05
    peers = [center + torch.randn(n_elems, generator=g) * 0.01 * (k + 1) for k in range(n_peers)]
    return center, peers, [float(w) for w in np.random.default_rng(0).dirichlet(np.ones(n_peers))]


def _sharded_worker(rank, world, port, n_peers, n_elems, root, q, hip):
    import os
    import sys

    for p in (os.path.join(root, "decentralized-learning_amd"), root, os.path.join(root, "tests")):
        sys.path.insert(0, p)
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), HSA_ENABLE_IPC_MODE_LEGACY="0")
    torch.set_num_threads(1)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from accdfl_amd.core.sharding import BucketShardedFedAvg

        center, peers, weights = _sharded_inputs(n_peers, n_elems)
        sh = BucketShardedFedAvg(n_elems, torch.float32, bounded=_hip_bounded() if hip else _oracle_bounded())
        s, e = sh.local_range

        def bucket(v):
            out = torch.zeros(sh.bucket_len)
            out[: e - s] = v[s:e]
            return out

        mine = sh.reduce_bucket_bounded([bucket(p) for p in peers], bucket(center), 0.02 * math.sqrt(n_elems), weights)
        q.put((rank, sh.all_gather(mine).numpy().copy()))
    finally:
        dist.destroy_process_group()


def run_sharded(world, n_peers, n_elems, hip=False):
    import os

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_sharded_worker, args=(r, world, port, n_peers, n_elems, root, q, hip)) for r in range(world)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=100) for _ in range(world))
    for p in procs:
        p.join(60)
        assert p.exitcode == 0
    center, peers, weights = _sharded_inputs(n_peers, n_elems)
    want, norms, added = no.bounded([[p] for p in peers], weights, [center], 0.02 * math.sqrt(n_elems))
    assert min(norms) < 0.02 * math.sqrt(n_elems) < max(norms)
    for r in range(world):
        no.assert_close(torch.from_numpy(got[r]), want[0], n_elems, added[0])


@pytest.mark.parametrize("world, n_peers, n_elems", [(2, 3, 1001), (3, 5, 130), (2, 4, 64)])
def test_sharded_bounded_over_gloo(world, n_peers, n_elems):
    """Every rank holds one bucket of every peer (an empty one at 64 elements); the norms are the whole model's."""
    run_sharded(world, n_peers, n_elems)
