"""Shaped attention and eviction without a GPU: intervals of masks, refusals ahead of any launch, sizes of workspaces."""
import ctypes as C
import os

import pytest
import torch

from smcsd_b200.ops import native as K
from smcsd_b200.ops import native_shaped as N

from shaped_oracle import choose

needs_library = pytest.mark.skipif(not os.path.exists(os.path.join(os.path.dirname(K.__file__), "libsmcsd_b200.so")), reason="kernel library not built")


@pytest.mark.parametrize("window", [0, 1, 4, 100])
@pytest.mark.parametrize("docs", [False, True])
@pytest.mark.parametrize("prefix", [None, 0, 1, 6, 50])
def test_score_bounds_against_the_masks_they_stand_for(window, docs, prefix):
    pos = torch.arange(23)
    doc = torch.tensor([0] * 5 + [1] * 1 + [2] * 10 + [3] * 7)
    starts = torch.tensor([0, 5, 6, 16])[doc]
    b = N.score_bounds(pos, window=window, doc_first=starts if docs else None, prefix=prefix)
    assert b.dtype == torch.int32 and b.shape == (23, 2)
    got = (pos >= b[:, :1]) & (pos <= b[:, 1:])
    want = pos <= pos[:, None]
    if prefix:
        want = want | ((pos < prefix) & (pos[:, None] < prefix))     # the tokens of the prefix see each other
    if window:
        want = want & (pos > pos[:, None] - window)
    if docs:
        want = want & (pos >= starts[:, None])
    assert torch.equal(got, want)


def test_score_bounds_takes_a_prefix_per_token():
    b = N.score_bounds(torch.tensor([0, 1, 5, 0, 1]), prefix=torch.tensor([2, 2, 2, 4, 4]))
    assert b.tolist() == [[0, 1], [0, 1], [0, 5], [0, 3], [0, 3]]


def test_choose_breaks_ties_to_the_lower_index_and_keeps_nan():
    assert choose([1.0, 1.0, 1.0, 1.0, 1.0, 1.0], 4, 1, 1) == [0, 1, 2, 5]
    assert choose([0.0, float("nan"), 5.0, 9.0, 1.0], 2, 0, 0) == [1, 3]
    assert choose([3.0, 2.0], 5, 1, 1) == [0, 1] and choose([3.0, 2.0, 9.0, 1.0], 2, 1, 1) == [0, 3]


def test_tensors_off_the_gpu_are_refused():
    z = torch.zeros(4, 64, dtype=torch.bfloat16)
    i = torch.zeros(4, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA device"):
        N.attention_shaped_prompt(z, z, z, i, i, z, T=4, Hq=1, Hkv=1, D=64, scale=0.125, status=i[0])
    with pytest.raises(ValueError, match="CUDA device"):
        N.evict_tokens(i, i[0], i[0], i[0], z.float().view(4, 1, 64), i[0], i[0], i[0], keep=1, first=0, last=0, kept=i, work=i[0].to(torch.uint8), status=i[0])


@needs_library
def test_workspaces():
    assert N.shaped_step_work_bytes(1, 1, 8, 8, 64) >= 4 * 32768
    small, large = N.shaped_step_work_bytes(4, 1, 32, 8, 128, 1000), N.shaped_step_work_bytes(4, 1, 32, 8, 128, 64000)
    assert large - small >= 63000 * 32 * 4 and large - small < 64500 * 32 * 4
    for bad in [(0, 1, 8, 8, 64), (1, 0, 8, 8, 64), (1, 1, 8, 3, 64), (1, 1, 8, 8, 96), (1, 65, 8, 8, 64), (1, 9, 64, 8, 64), (1025, 1, 8, 8, 64), (1024, 1, 64, 64, 64)]:
        with pytest.raises(ValueError, match="no step"):
            N.shaped_step_work_bytes(*bad)
    assert N.evict_work_bytes(1000) >= 1001 // 8


@needs_library
def test_entries_refuse_on_the_host():
    """Sizes, alignments and options that the kernels do not take: an error code ahead of any launch."""
    L, p = N._library(), 1 << 20

    def prompt(q=p, ldq=512, k=p, v=p, runs=p, out=p, ldo=512, Hq=8, Hkv=2, D=64, scale=0.125, cap=0.0, bounds=None):
        return L.smc_shaped_prompt(q, ldq, k, v, 7, p, 8, 1, None, 0, runs, 1, out, ldo, None, 4, Hq, Hkv, D, scale, cap, None, bounds, p, 0, None)
    for name in ("q", "k", "v", "runs", "out"):
        assert prompt(**{name: p + 8}) == -141, name
    assert prompt(ldq=516) == prompt(ldo=516) == prompt(bounds=p + 4) == -142
    assert prompt(D=96) == prompt(Hq=9) == prompt(Hkv=0) == prompt(Hq=258) == -140
    for bad in (dict(cap=-1.0), dict(cap=float("nan")), dict(cap=float("inf")), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan"))):
        assert prompt(**bad) == -143, bad

    def mass(q=p, k=p, runs=p, stride=8, Hq=8, Hkv=2, D=64, scale=0.125, cap=0.0):
        return L.smc_shaped_mass(q, 512, k, 7, p, 8, 1, None, 0, runs, 1, p, p, stride, 4, Hq, Hkv, D, scale, cap, None, None, p, 0, None)
    assert mass(q=p + 8) == mass(k=p + 8) == mass(runs=p + 8) == -161
    assert mass(D=32) == mass(Hq=7) == -160 and mass(scale=0.0) == mass(cap=-2.0) == -162 and mass(stride=7) == -163

    def step(q=p, k=p, work=p, nbytes=1 << 30, m=None, stride=8, bs=2, E=1, Hq=8, Hkv=2, D=64, scale=0.125):
        return L.smc_shaped_step(q, 512, k, p, 7, p, 8, 1, None, 0, p, p, p, 512, None, m, stride, bs, E, Hq, Hkv, D, scale, 0.0, None, None, work, nbytes, p, 0, None)
    assert step(q=p + 2) == step(k=p + 8) == step(work=p + 8) == -151
    assert step(D=80) == step(E=17) == step(bs=2000) == -150 and step(scale=0.0) == -152
    assert step(m=p, stride=7) == -153 and step(nbytes=1000) == -154
    assert step(m=p, nbytes=N.shaped_step_work_bytes(2, 1, 8, 2, 64)) == -154      # no room for the scores of a single tile

    def evict(stride=64, kps=64, ms=64, heads=2, keep=8, first=1, last=1, kept=p, work=p, nbytes=1 << 20, rows=3):
        return L.smc_evict(p, stride, p, kps, p, ms, p, 4, p, p, rows, heads, keep, first, last, kept, p, p, p, 100, work, nbytes, p, None)
    assert evict(keep=0) == evict(first=-1) == evict(last=8) == evict(first=9) == evict(heads=0) == evict(kept=None) == evict(rows=5000) == -170
    assert evict(stride=1 << 20, ms=1 << 20, kps=1 << 20) == evict(ms=63) == evict(kps=63) == -171
    assert evict(nbytes=100) == evict(work=p + 2) == -172
