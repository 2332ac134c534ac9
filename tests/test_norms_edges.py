"""The norm operators' rules at their edges, for what needs no GPU: which views overlap, how large a launch is, and the
staging of rounds of CPU models."""
import itertools
import os
import random
import subprocess

import pytest
import torch


def _bytes_of(t):
    size = t.element_size()
    return [t.data_ptr() + size * sum(i * st for i, st in zip(at, t.stride())) + b
            for at in itertools.product(*[range(n) for n in t.shape]) for b in range(size)]


def test_overlaps_are_told_from_neighbours():
    """Random views of one buffer, of three element sizes, against their bytes."""
    from accdfl_amd.core.norms import _Elements

    buf = torch.zeros(400)
    bases = [buf, buf.view(torch.int16), buf.view(torch.int64)]
    rng = random.Random(1)

    def view():
        axes, times = rng.randint(0, 3), rng.choice([1, 1, 2, 3, 4])
        return rng.choice(bases).as_strided([rng.randint(1, 4) for _ in range(axes)],
                                            [times * rng.randint(0, 5) for _ in range(axes)], rng.randint(0, 60))
    met = itself = 0
    for _ in range(4000):
        a, b = view(), view()
        ba, bb = _bytes_of(a), _bytes_of(b)
        assert _Elements.of(a).meets_itself() == (len(set(ba)) < len(ba)), (a.shape, a.stride())
        assert _Elements.of(a).meet(_Elements.of(b)) == bool(set(ba) & set(bb)), (a.shape, a.stride(), b.shape, b.stride())
        met += bool(set(ba) & set(bb))
        itself += len(set(ba)) < len(ba)
    assert met > 300 and itself > 300


def test_refusals_of_views_by_their_elements():
    from accdfl_amd import _lib
    from accdfl_amd.core.norms import _refuse_overlaps

    m = torch.zeros(10, 12)
    fresh = torch.zeros(10, 3)
    fine = [
        ([m[:, :3], m[:, 3:6]], [m[:, :3], m[:, 3:6]]),            # in place
        ([fresh, fresh], [m[:, :3], m[:, 3:6]]),                   # an input twice
        ([m[:, 6:9], m[:, 6:9]], [m[:, :3], m[:, 3:6]]),           # in the gaps of the outputs
        ([torch.zeros(0)], [m[:0, 0]]),
    ]
    for ins, outs in fine:
        _refuse_overlaps([ins, outs], ["tensors", "outs"], 1)
    for ins, outs, what in (
            ([fresh, fresh], [m[:, :3], m[:, 2:5]], "outs tensor [01] overlaps outs tensor [01]"),
            ([fresh, fresh], [m[:, :3], m[:, :3]], "outs tensor [01] overlaps outs tensor [01]"),
            ([m[:, 3:6], m[:, :3]], [m[:, :3], m[:, 3:6]], "tensors tensor 0 overlaps outs tensor 1"),
            ([m[:, 1:4]], [m[:, :3]], "tensors tensor 0 overlaps outs tensor 0"),
            ([m[:5, :5]], [m[:5, :5].t()], "tensors tensor 0 overlaps outs tensor 0")):
        with pytest.raises(_lib.DlaggError, match=what):
            _refuse_overlaps([ins, outs], ["tensors", "outs"], 1)
    for out in (m[:, :1].expand(10, 3), m.as_strided((3, 3), (1, 1)), m.as_strided((5, 4), (3, 4))):
        with pytest.raises(ValueError, match="outs tensor 0: an output has elements that share memory"):
            _refuse_overlaps([[torch.zeros(out.shape)], [out]], ["tensors", "outs"], 1)


def test_no_launch_has_more_threads_than_hip_takes(tmp_path):
    """The grid of the kernels that give each unit a workgroup: an average of 64 GiB (2^26 units of 64 threads), a clip of
    256 GiB (2^24 units of 256) and everything around them."""
    from accdfl_amd import _lib

    src = tmp_path / "grid.cpp"
    src.write_text("""
#include "dlagg_internal.h"
#include <cstdio>
#include <cstdlib>
int main(int n, char** v) {
  for (int i = 1; i + 1 < n; i += 2) std::printf("%lld\\n", (long long)dla_internal_grid(std::atoll(v[i]), std::atoi(v[i + 1])));
}
""")
    exe = str(tmp_path / "grid")
    subprocess.run(["g++", "-std=c++17", "-I", os.path.dirname(_lib.CSRC_INTERNAL), "-o", exe, str(src)], check=True)
    asked = [(units, threads) for threads in (64, 256) for power in (0, 10, 23, 24, 25, 26, 27, 31, 32, 53)
             for units in (2 ** power - 1, 2 ** power, 2 ** power + 1)]
    out = subprocess.run([exe] + [str(v) for pair in asked for v in pair], check=True, capture_output=True, text=True)
    for (units, threads), grid in zip(asked, map(int, out.stdout.split())):
        assert grid * threads < 2 ** 32 and grid <= units, (units, threads, grid)
        assert grid == units or (grid + 1) * threads >= 2 ** 32, (units, threads, grid)


def test_stages_of_rounds_at_once(monkeypatch):
    """A round that begins within another one, in any thread, has a stage of its own; they are kept for later rounds, but
    not that of a round that failed."""
    from accdfl_amd.core.gradient_aggregation import norm_bounded as nb

    monkeypatch.setattr(nb, "_HostStage", lambda device: object())
    monkeypatch.setattr(nb, "_free_stages", {})
    with nb._host_stage(0) as a:
        with nb._host_stage(0) as b, nb._host_stage(1) as c:
            assert len({id(a), id(b), id(c)}) == 3
    with nb._host_stage(0) as first, nb._host_stage(0) as second:
        assert {id(first), id(second)} == {id(a), id(b)}
        nb.release_staging()
    assert len(nb._free_stages[0]) == 2 and 1 not in nb._free_stages
    with pytest.raises(ZeroDivisionError):
        with nb._host_stage(0):
            1 / 0
    assert len(nb._free_stages[0]) == 1
