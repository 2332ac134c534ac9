"""FedAvg of norm-bounded updates: an aggregator that one peer cannot move further than a bound.

FedAvg averages whatever arrived (accdfl/core/gradient_aggregation/fedavg.py:20-25): one peer that sends a model
far from the others, or NaNs, moves or destroys the result.  Here every peer's update — its model minus a centre,
over all parameters together — is scaled to a norm of at most ``max_norm`` before it is averaged, and a peer whose
update is not finite adds nothing::

    n_k    = || p_k - c ||_2
    result = c + sum_k w_k min(1, max_norm / n_k) (p_k - c)

With a bound above every norm and weights that add up to 1 this is the weighted average of the models, carried in
64 bits and rounded once (FedAvg rounds every step, as the reference does).

The contract is FedAvg.aggregate's (weights, defaults, errors; the result is ``copy.deepcopy(models[0])`` with
the averaged parameters, on models[0]'s device), selected by ``settings.gradient_aggregation =
GradientAggregationMethod.NORM_BOUNDED_FEDAVG`` with ``settings.max_update_norm``.  Stricter than FedAvg: the models
and the centre must have the same parameters (count, shapes, dtypes).
"""
from __future__ import annotations

from typing import List, Optional

import torch
from torch import nn

from accdfl_amd import _lib
from accdfl_amd.core import norms as _norms
from accdfl_amd.core import wsum as _wsum
from accdfl_amd.core.gradient_aggregation import GradientAggregation
from accdfl_amd.core.gradient_aggregation import fedavg as _fedavg


def _device_round(models: List[nn.Module], weights, center: nn.Module, max_norm: float) -> Optional[nn.Module]:
    """The round of device-resident models of one layout: the centre and the models walked in one pass, the
    result's parameters made around the launches as FedAvg's device round makes them.  None when the models do
    not qualify (the general path then handles the round)."""
    mod = _lib.walk_module()
    if mod is None:
        return None
    everything = [center] + models
    tables = mod.module_tables(everything, _fedavg._PLAIN_SET)
    if tables is None:
        # classes not met before are classified once, as FedAvg's layout does it
        fresh = {type(sub) for m in (center, models[0]) for sub in m.modules()} - _fedavg._plain_walk_cls.keys()
        if any([_fedavg._plain_walk(cls) for cls in fresh]):
            tables = mod.module_tables(everything, _fedavg._PLAIN_SET)
    if tables is None:
        return None
    objs = mod.tensors(models[0], _fedavg._PLAIN_SET)
    if objs is None or any([type(p) is not nn.Parameter for p in objs[0]]):
        return None
    p0, b0 = objs
    memo = {}
    with _norms._place(torch.device("cuda", tables.device), None):
        blocks, outs = mod.param_blocks(p0)
        _norms.wsum_bounded_tables(tables, outs, weights, max_norm)
        # while the round runs: the parameters' Python objects, models[0]'s buffers, the module tree
        mod.param_wrap(blocks, p0, memo)
        _fedavg._seed_buffers(b0, memo)
        return _fedavg._clone_value(models[0], memo)


def _check_layout(models: List[nn.Module], center: nn.Module) -> List[List[torch.Tensor]]:
    """The parameters of the centre and of every model; raises unless all have models[0]'s."""
    lists = [_fedavg._parameters(m) for m in [center] + models]
    first = lists[1]
    for ps, name in zip(lists, ["center"] + ["model %d" % k for k in range(len(models))]):
        if len(ps) != len(first):
            raise RuntimeError("NormBoundedFedAvg: %s has %d parameters, model 0 has %d" % (name, len(ps), len(first)))
        for i, (p, q) in enumerate(zip(ps, first)):
            _wsum.dtype_code(p.dtype)
            if p.shape != q.shape or p.dtype != q.dtype:
                raise RuntimeError("NormBoundedFedAvg: parameter %d of %s is %s %s, model 0 has %s %s"
                                   % (i, name, p.dtype, tuple(p.shape), q.dtype, tuple(q.shape)))
    return lists


def _general_round(models: List[nn.Module], weights, center: nn.Module, max_norm: float) -> nn.Module:
    """Any other round (CPU models, models on several devices, parameters of several dtypes): everything is
    brought to models[0]'s GPU (the current one for CPU models), averaged there and copied into the result."""
    lists = _check_layout(models, center)
    result = _fedavg._center_copy(models[0])
    params = list(result.parameters())
    if not params:
        return result
    home = params[0].device
    device = _wsum.require_device(home if home.type == "cuda" else None)
    if len({p.dtype for p in params}) == 1 and all(p.device.type == "cpu" for ps in lists for p in ps):
        from accdfl_amd.core.peer_slab import PeerSlab

        slab = PeerSlab([p.shape for p in params], params[0].dtype, len(models), device)
        for ps in lists[1:]:
            slab.stage(ps)
        slab.reduce_bounded_into(params, max_norm, weights, center=None if center is models[0] else lists[0])
        return result
    resident = [[p.detach().to(device) for p in ps] for ps in lists]
    outs = [torch.empty_like(p) for p in resident[0]]
    _norms.wsum_bounded_multi(resident[1:], weights, resident[0], max_norm, outs)
    for p, o in zip(params, outs):
        p.copy_(o)
    return result


class NormBoundedFedAvg(GradientAggregation):
    """``NormBoundedFedAvg(max_norm, center).aggregate(models, weights)``.  ``center``: the model the updates are
    measured from — the one the round started from; default models[0], the local model of a gossip merge."""

    def __init__(self, max_norm: float, center: Optional[nn.Module] = None):
        self.max_norm = _norms._bound(max_norm)
        self.center = center

    def aggregate(self, models: List[nn.Module], weights: List[float]):
        if not weights:
            weights = [float(1. / len(models)) for _ in range(len(models))]
        else:
            assert len(weights) == len(models)
        weights = [float(w) for w in weights]
        models = list(models)
        _norms._check_peers(len(models))
        with torch.no_grad():
            center = self.center if self.center is not None else models[0]
            done = _device_round(models, weights, center, self.max_norm)
            return done if done is not None else _general_round(models, weights, center, self.max_norm)
