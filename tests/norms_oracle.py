"""The norm and clipping operators from their definitions, in 64 bits on the CPU (test infrastructure only), and how
far a correct result may be from them.

Norms, products and averages are carried in 64 bits and rounded once (16-bit types through float32), so with u = eps / 2
of the storage type, v = 2^-24 (0 for float64) and w = 2^-53 * terms for the 64-bit sums,
    |got - want| <= (u + v) |want| + w * (sum of the magnitudes added) + half the smallest subnormal.
The averages of 16-bit types are carried in 32 bits: c + sum_k a_k d_k over N peers rounds a_k and d_k once each (2 * 2^-24 of
|a_k d_k|), every one of the N fused additions (2^-24 of a partial sum, at most M = |c| + sum_k |a_k d_k|) and the
addition of c (2^-24 M): at most (N + 3) 2^-24 M, beside the terms above."""
import math

import numpy as np
import torch

CLIP_EPS = 1e-6


def wide(t):
    return t.detach().cpu().to(torch.float64).reshape(-1)


def norm(tensors, p=2.0):
    vs = [wide(t) for t in tensors if t.numel()]
    if not vs:
        return 0.0
    v = torch.cat(vs).numpy()
    with np.errstate(all="ignore"):
        if p == math.inf:
            return float(np.max(np.abs(v)))
        return float(np.sum(np.abs(v))) if p == 1.0 else float(np.sqrt(np.sum(np.square(v))))


def ratio(n, max_norm):
    with np.errstate(all="ignore"):
        q = np.float64(max_norm) / (np.float64(n) + CLIP_EPS)
    return float(1.0 if q > 1.0 else q)


def clip(tensors, max_norm, p=2.0):
    n = norm(tensors, p)
    r = ratio(n, max_norm)
    return [t.detach().cpu().to(torch.float64) * r for t in tensors], n


def update_norms(models, center):
    return [norm([m.detach().cpu().to(torch.float64) - c.detach().cpu().to(torch.float64) for m, c in zip(ms, center)])
            for ms in models]


def shares(norms, weights, max_norm):
    return [w * (1.0 if n <= max_norm else max_norm / n) if math.isfinite(n) else 0.0 for n, w in zip(norms, weights)]


def bounded(models, weights, center, max_norm, norms=None):
    """(results, norms, (N + 3) M for each result)."""
    if norms is None:
        norms = update_norms(models, center)
    outs, added = [], []
    for i, c in enumerate(center):
        c = c.detach().cpu().to(torch.float64)
        acc, mag = torch.zeros_like(c), c.abs()
        for ms, a, n in zip(models, shares(norms, weights, max_norm), norms):
            if a == 0.0 or not math.isfinite(n):
                continue
            d = a * (ms[i].detach().cpu().to(torch.float64) - c)
            acc, mag = acc + d, mag + d.abs()
        outs.append(c + acc)
        added.append(mag * (len(models) + 3))
    return outs, norms, added


def assert_norm(got, want, terms):
    got = got.detach().cpu()
    want = np.atleast_1d(np.asarray(want, dtype=np.float64))
    g = np.atleast_1d(got.numpy().astype(np.float64))
    assert g.shape == want.shape
    u = torch.finfo(got.dtype).eps / 2
    tol = (u + 2.0 ** -53 * (terms + 8)) * np.abs(want)
    for a, b, t in zip(g, want, tol):
        if math.isfinite(b):
            assert math.isfinite(a) and abs(a - b) <= t + 2.0 ** -150, (a, b, abs(a - b), t)
        else:
            assert (math.isnan(a) and math.isnan(b)) or a == b, (a, b)


def assert_close(got, want, terms, added=None):
    """``got`` in its storage type against ``want`` in 64 bits; ``terms``: elements behind the norm in it."""
    info = torch.finfo(got.dtype)
    g = got.detach().cpu().to(torch.float64)
    assert g.shape == want.shape
    # beyond the type's largest value by half a step: infinite
    v = 0.0 if got.dtype == torch.float64 else 2.0 ** -24
    mag = want.abs() if added is None else added
    tol = (info.eps / 2 + v) * want.abs() + 2.0 ** -53 * (terms + 16) * mag + info.smallest_normal * info.eps / 2
    if added is not None and got.dtype in (torch.bfloat16, torch.float16):
        tol = tol + 2.0 ** -24 * added
    fine = torch.isfinite(want) & (want.abs() <= info.max)
    bad = fine & ~((g - want).abs() <= tol)
    assert not bool(bad.any()), "%d of %d differ, worst %g at tolerance %g" % (
        int(bad.sum()), g.numel(), float((g - want).abs()[bad].max()), float(tol[bad].max()))
    nan = torch.isnan(want)
    assert bool((torch.isnan(g) == nan).all())
    inf = torch.isinf(want)
    assert bool((g[inf] == want[inf]).all())
