"""Shaped attention over the paged cache, key mass and eviction on the GPU against float64 (shaped_oracle.py)."""
import math

import pytest
import torch

from shaped_oracle import Cache, attend, choose, head_sums

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _N():
    from smcsd_b200.ops import native_shaped as N
    return N


def _status():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def _slopes(Hq):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], device=DEV)


def _bounds(kind, cache, runs, T):
    """Intervals of a mask for every query token; ``holes`` leaves some tokens without a key."""
    if kind == "causal":
        return None
    b = torch.zeros(T, 2, dtype=torch.int32, device=DEV)
    for row, held, at, n in runs:
        pos = cache.positions(row)
        own = torch.cat([torch.full((max(0, -held),), -1, device=DEV), pos[max(held, 0):]])
        N = _N()
        if kind == "window":
            b[at:at + n] = N.score_bounds(own, window=7)
        elif kind == "documents":
            b[at:at + n] = N.score_bounds(own, doc_first=own.clamp(min=0) // 13 * 13)
        elif kind == "prefix":
            b[at:at + n] = N.score_bounds(own, prefix=40)
        else:
            b[at:at + n] = N.score_bounds(own, window=50)
            b[at:at + n:3] = torch.tensor([9, 8], device=DEV).int()                    # first behind last
    return b


def _tolerances(cache, q, Hq, scale, softcap):
    """Outputs: a probability and an output are each rounded to eight bits once, at most half a step 2^-9 of the values' range each; sums of |q||k| in fp32 are off
    by 2^-24 per product and a capped score by 2.8e-6 of itself, which moves a probability by as much.  lse: those two."""
    big = float((q.double().view(-1, cache.D).norm(dim=1).max() * cache.k[1:].double().view(-1, cache.D).norm(dim=1).max()) * scale) if len(cache.k) > 1 else 0.0
    score = min(big, softcap or big)
    moved = cache.D * 2.0 ** -24 * big + 3e-6 * score + 1e-6
    vmax = float(cache.v[1:].double().abs().max()) if len(cache.v) > 1 else 0.0
    return (2 * 2.0 ** -9 + 2 * moved) * vmax, moved + 2.0 ** -22 * (score + 12)


def _check(got, want, lse, want_lse, cache, q, Hq, scale, softcap):
    tol, tol_lse = _tolerances(cache, q, Hq, scale, softcap)
    assert float((got.double().view(want.shape) - want).abs().max()) <= tol
    assert torch.equal(torch.isinf(lse), torch.isinf(want_lse))
    there = torch.isfinite(want_lse)
    assert float((lse.double() - want_lse)[there].abs().max() if bool(there.any()) else 0.0) <= tol_lse
    assert not bool(got.view(want.shape)[~there].any())                                # nothing visible: zeros


HEADS = [(32, 8, 64), (14, 2, 64), (4, 4, 128), (16, 4, 128), (8, 1, 128), (16, 2, 256), (3, 1, 256)]
RUNS = {"one": [(0, 1)], "edges": [(0, 63), (0, 64), (5, 65), (127, 1), (128, 129), (300, 2), (0, 0)], "long": [(0, 700), (513, 130)]}


def _prompt(cache, sizes):
    runs, at = [], 0
    for i, (held, n) in enumerate(sizes):
        runs.append((i + 1, held, at, n))
        at += n
    return runs, at


@pytest.mark.parametrize("mask", ["causal", "window", "documents", "prefix", "holes"])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("sizes,order,shed,softcap,alibi", [("one", "up", False, 0.0, True), ("edges", "scattered", True, 30.0, False), ("edges", "up", False, 0.0, False),
                                                            ("long", "down", True, 0.0, True), ("long", "up", False, 5.0, True)])
def test_prompt_attention(Hq, Hkv, D, mask, sizes, order, shed, softcap, alibi):
    N = _N()
    c = Cache([a + n for a, n in RUNS[sizes]], Hkv, D, seed=D + Hq, order=order, shed=shed)
    runs, T = _prompt(c, RUNS[sizes])
    q = (1.7 * torch.randn(T, Hq * D, device=DEV, generator=torch.Generator(DEV).manual_seed(3))).bfloat16()
    scale, slopes, bounds = D ** -0.5, _slopes(Hq) if alibi else None, _bounds(mask, c, runs, T)
    want, want_lse, mass = attend(c, runs, q, Hq, scale=scale, softcap=softcap, slopes=slopes, bounds=bounds)
    # queries and outputs inside wider rows, rows behind the last token
    wide, out = torch.zeros(T, Hq * D + 24, dtype=torch.bfloat16, device=DEV), torch.full((T + 3, Hq * D + 8), 7.0, dtype=torch.bfloat16, device=DEV)
    wide[:, 16:16 + Hq * D] = q
    lse, st = torch.full((T, Hq), 5.0, device=DEV), _status()
    dev_runs = torch.tensor(runs, dtype=torch.int32, device=DEV)
    shape = dict(T=T, Hq=Hq, Hkv=Hkv, D=D, scale=scale, status=st, softcap=softcap, slopes=slopes, bounds=bounds, key_pos=c.key_pos)
    N.attention_shaped_prompt(wide[:, 16:16 + Hq * D], c.k, c.v, c.table, dev_runs, out[:, :Hq * D], lse=lse, **shape)
    torch.cuda.synchronize()
    assert int(st) == 0
    _check(out[:T, :Hq * D], want, lse, want_lse, c, q, Hq, scale, softcap)
    assert bool((out[T:] == 7.0).all()) and bool((out[:, Hq * D:] == 7.0).all())
    # the mass of the same tokens, on top of what is there
    m = torch.rand(c.table.shape[0], Hkv, c.table.shape[1] + 3, device=DEV)
    before = m.clone()
    N.attention_key_mass(wide[:, 16:16 + Hq * D], c.k, c.table, dev_runs, lse, m, **shape)
    torch.cuda.synchronize()
    assert int(st) == 0
    moved = _tolerances(c, q, Hq, scale, softcap)[1] * 2                               # score and lse, each as far off as an lse may be
    for row, held, at, n in runs:
        w = mass[row]
        diff = (m[row, :, :w.shape[1]].double() - before[row, :, :w.shape[1]].double() - w).abs()
        assert bool((diff <= moved * w + 2.0 ** -22 * (w + 1)).all())                  # and one fp32 addition to numbers below one
        assert torch.equal(m[row, :, w.shape[1]:], before[row, :, w.shape[1]:])
    assert torch.equal(m[0], before[0])


def test_prompt_attention_of_many_sequences_and_far_positions():
    """More sequences than a warp has lanes, most of a few tokens; positions up to 2^24 in a thinned-out cache; scores far beyond the polynomial's reach."""
    N = _N()
    sizes = [(i % 5 * 40, 1 + i * 7 % 23) for i in range(75)] + [(2000, 40)]
    c = Cache([a + n for a, n in sizes], 2, 64, shed=True, seed=9)
    c.key_pos[1:] += (1 << 24) - 20000
    runs, T = _prompt(c, sizes)
    q, st = (25 * torch.randn(T, 8 * 64, device=DEV)).bfloat16(), _status()
    slopes = _slopes(8)
    b = torch.stack([torch.zeros(T, device=DEV), torch.full((T,), 2.0 ** 31 - 1, device=DEV)], 1).to(torch.int64).clamp(max=2 ** 31 - 1).int()    # everything
    for bounds in (None, b):
        want, want_lse, _ = attend(c, runs, q, 8, scale=0.125, softcap=20.0, slopes=slopes, bounds=bounds)
        out, lse = torch.zeros(T, 512, dtype=torch.bfloat16, device=DEV), torch.zeros(T, 8, device=DEV)
        N.attention_shaped_prompt(q, c.k, c.v, c.table, torch.tensor(runs, dtype=torch.int32, device=DEV), out, T=T, Hq=8, Hkv=2, D=64, scale=0.125, status=st, softcap=20.0,
                                  slopes=slopes, bounds=bounds, key_pos=c.key_pos, lse=lse)
        torch.cuda.synchronize()
        assert int(st) == 0
        _check(out, want, lse, want_lse, c, q, 8, 0.125, 20.0)


@pytest.mark.parametrize("Hq,Hkv,D", [(128, 1, 64), (100, 1, 128), (65, 1, 256), (66, 2, 64)])
def test_groups_that_fill_or_miss_a_tile(Hq, Hkv, D):
    """One token or two to a tile of rows, with rows left over."""
    N = _N()
    c = Cache([150, 3], Hkv, D, shed=True)
    runs, T = [(1, 130, 0, 20), (2, 0, 20, 3)], 23
    q, st = torch.randn(T, Hq * D, device=DEV).bfloat16(), _status()
    want, want_lse, mass = attend(c, runs, q, Hq, scale=D ** -0.5, softcap=20.0, slopes=_slopes(Hq))
    out, lse, m = torch.zeros(T, Hq * D, dtype=torch.bfloat16, device=DEV), torch.zeros(T, Hq, device=DEV), torch.zeros(3, Hkv, c.table.shape[1], device=DEV)
    kw = dict(T=T, Hq=Hq, Hkv=Hkv, D=D, scale=D ** -0.5, status=st, softcap=20.0, slopes=_slopes(Hq), key_pos=c.key_pos)
    r = torch.tensor(runs, dtype=torch.int32, device=DEV)
    N.attention_shaped_prompt(q, c.k, c.v, c.table, r, out, lse=lse, **kw)
    N.attention_key_mass(q, c.k, c.table, r, lse, m, **kw)
    torch.cuda.synchronize()
    assert int(st) == 0
    _check(out, want, lse, want_lse, c, q, Hq, D ** -0.5, 20.0)
    moved = _tolerances(c, q, Hq, D ** -0.5, 20.0)[1] * 2
    for row, w in mass.items():
        assert bool(((m[row, :, :w.shape[1]].double() - w).abs() <= moved * w + 2.0 ** -22 * (w + 1)).all())


@pytest.mark.parametrize("slope", [0.9, -0.002])
def test_distance_bias_against_opposed_scores(slope):
    """The highest scores lie far away and the distance takes them back (or adds to them): the reference must not bury the row."""
    N = _N()
    c = Cache([400], 1, 64, order="up")
    c.k[1:] = 0
    c.k[1:, 0] = torch.linspace(200, -200, 400, device=DEV).bfloat16()
    q, st = torch.zeros(400, 64, dtype=torch.bfloat16, device=DEV), _status()
    q[:, 0] = 8.0
    slopes = torch.tensor([slope], device=DEV)
    for cap in (0.0, 150.0):
        want, want_lse, _ = attend(c, [(1, 0, 0, 400)], q, 1, scale=0.125, softcap=cap, slopes=slopes)
        out, lse = torch.zeros_like(q), torch.zeros(400, 1, device=DEV)
        N.attention_shaped_prompt(q, c.k, c.v, c.table, torch.tensor([[1, 0, 0, 400]], dtype=torch.int32, device=DEV), out, T=400, Hq=1, Hkv=1, D=64, scale=0.125, status=st,
                                  softcap=cap, slopes=slopes, lse=lse)
        torch.cuda.synchronize()
        assert int(st) == 0
        _check(out, want, lse, want_lse, c, q, 1, 0.125, cap)


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 32, 8), (128, 16, 4), (256, 16, 2)])
def test_prompt_bits_do_not_depend_on_pages_or_neighbours(D, Hq, Hkv):
    """The same keys in ascending and scattered pages, alone and beside another sequence: the same bits."""
    N = _N()
    outs, st, n = [], _status(), 300
    q = torch.randn(n, Hq * D, device=DEV).bfloat16()
    k, v = (torch.randn(n, Hkv * D, device=DEV).bfloat16() for _ in range(2))
    for order, more in (("up", 0), ("scattered", 0), ("up", 90)):
        c = Cache([n] + [more] * (more > 0), Hkv, D, order=order)
        pages = c.table[1, :n].long()
        c.k[pages], c.v[pages] = k, v
        runs = [[1, 0, 0, n]] + [[2, 0, n, more]] * (more > 0)
        qq = torch.cat([q, q[:more]])
        out = torch.zeros_like(qq)
        N.attention_shaped_prompt(qq, c.k, c.v, c.table, torch.tensor(runs, dtype=torch.int32, device=DEV), out, T=n + more, Hq=Hq, Hkv=Hkv, D=D, scale=D ** -0.5, status=st,
                                  softcap=30.0)
        outs.append(out[:n])
    torch.cuda.synchronize()
    assert int(st) == 0 and torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


STEPS = {"one": [1], "short": [3, 1, 0, 2, 70, 5], "ragged": [64, 65, 1, 700, 129, 2500, 31, 4], "long": [9000]}


@pytest.mark.parametrize("mask", ["causal", "window", "documents", "prefix", "holes"])
@pytest.mark.parametrize("Hq,Hkv,D,E", [(32, 8, 64, 1), (14, 2, 64, 1), (32, 8, 64, 9), (4, 4, 128, 3), (16, 4, 128, 4), (32, 8, 128, 9), (8, 1, 128, 8), (16, 2, 256, 1), (16, 2, 256, 2),
                                        (16, 2, 256, 8), (5, 1, 256, 5)])
@pytest.mark.parametrize("lens,shed,softcap,alibi", [("one", False, 0.0, True), ("short", True, 30.0, False), ("ragged", True, 0.0, True), ("ragged", False, 5.0, True),
                                                     ("long", False, 0.0, False)])
def test_step_attention_with_mass(Hq, Hkv, D, E, mask, lens, shed, softcap, alibi):
    N = _N()
    c = Cache(STEPS[lens], Hkv, D, seed=D + E, shed=shed)
    bs = len(c.lens)
    runs = [(i + 1, n - E, i * E, E) for i, n in enumerate(c.lens)]
    q = (1.7 * torch.randn(bs * E, Hq * D, device=DEV, generator=torch.Generator(DEV).manual_seed(4))).bfloat16()
    scale, slopes, bounds = D ** -0.5, _slopes(Hq) if alibi else None, _bounds(mask, c, runs, bs * E)
    want, want_lse, mass = attend(c, runs, q, Hq, scale=scale, softcap=softcap, slopes=slopes, bounds=bounds)
    out, lse, st = torch.full((bs * E + 2, Hq * D + 8), 7.0, dtype=torch.bfloat16, device=DEV), torch.zeros(bs * E, Hq, device=DEV), _status()
    work = torch.zeros(N.shaped_step_work_bytes(bs, E, Hq, Hkv, D, sum(c.lens)), dtype=torch.uint8, device=DEV)
    m = torch.rand(c.table.shape[0], Hkv, c.table.shape[1], device=DEV)
    before = m.clone()
    rows, ln = torch.arange(1, bs + 1, device=DEV).int(), torch.tensor(c.lens, device=DEV).int()
    shape = dict(bs=bs, E=E, Hq=Hq, Hkv=Hkv, D=D, scale=scale, status=st, work=work, softcap=softcap, slopes=slopes, bounds=bounds, key_pos=c.key_pos)
    N.attention_shaped_step(q, c.k, c.v, c.table, rows, ln, out[:, :Hq * D], lse=lse, mass=m, **shape)
    torch.cuda.synchronize()
    assert int(st) == 0
    _check(out[:bs * E, :Hq * D], want, lse, want_lse, c, q, Hq, scale, softcap)
    assert bool((out[bs * E:] == 7.0).all()) and bool((out[:, Hq * D:] == 7.0).all())
    moved = _tolerances(c, q, Hq, scale, softcap)[1] * 2
    for row in range(1, bs + 1):
        w = mass[row]
        diff = (m[row, :, :w.shape[1]].double() - before[row, :, :w.shape[1]].double() - w).abs()
        assert bool((diff <= moved * w + 2.0 ** -22 * (w + 1)).all())
        assert torch.equal(m[row, :, w.shape[1]:], before[row, :, w.shape[1]:])
    # again, without mass and lse, in the same workspace: the same bits
    again = torch.zeros(bs * E, Hq * D, dtype=torch.bfloat16, device=DEV)
    N.attention_shaped_step(q, c.k, c.v, c.table, rows, ln, again, **shape)
    assert torch.equal(again, out[:bs * E, :Hq * D].contiguous())


def test_one_workspace_serves_batches_of_all_shapes():
    """Large and small batches by turns, captured into graphs that share the workspace, replayed in another order and on another stream."""
    N = _N()
    st, cases, graphs = _status(), [], []
    work = torch.zeros(N.shaped_step_work_bytes(40, 9, 32, 8, 128, 40 * 300), dtype=torch.uint8, device=DEV)
    for Hq, Hkv, D, E, lens in ((32, 8, 128, 9, [37 + 7 * i for i in range(40)]), (8, 2, 64, 1, [5000]), (32, 8, 128, 1, [300, 1, 900]), (16, 2, 256, 2, [77] * 9)):
        c = Cache(lens, Hkv, D, seed=E)
        q = torch.randn(len(lens) * E, Hq * D, device=DEV).bfloat16()
        want, _, mass = attend(c, [(i + 1, n - E, i * E, E) for i, n in enumerate(lens)], q, Hq, scale=D ** -0.5)
        m, out = torch.zeros(c.table.shape[0], Hkv, c.table.shape[1], device=DEV), torch.zeros_like(q)
        args = (q, c.k, c.v, c.table, torch.arange(1, len(lens) + 1, device=DEV).int(), torch.tensor(lens, device=DEV).int(), out)
        kw = dict(bs=len(lens), E=E, Hq=Hq, Hkv=Hkv, D=D, scale=D ** -0.5, status=st, work=work, mass=m)
        N.attention_shaped_step(*args, **kw)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            N.attention_shaped_step(*args, **kw)
        graphs.append(g)
        cases.append((c, want, mass, m, out, args, kw))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for i in (2, 0, 3, 1, 0, 2):
            graphs[i].replay()
    side.synchronize()
    assert int(st) == 0
    for i, (c, want, mass, m, out, args, kw) in enumerate(cases):
        assert float((out.double().view(want.shape) - want).abs().max()) <= _tolerances(c, args[0], kw["Hq"], kw["scale"], 0.0)[0]
        times = 1 + (2, 1, 2, 1)[i]
        for row, w in mass.items():
            assert float((m[row, :, :w.shape[1]].double() / times - w).abs().max()) < 1e-4 * float(w.max())


def test_calls_that_start_before_the_one_ahead_has_ended():
    """The same bits with programmatic launches, each call reading what the one ahead of it writes."""
    N = _N()
    Hq, Hkv, D, n = 16, 4, 128, 700
    c = Cache([n, 40], Hkv, D, shed=True)
    q, st = torch.randn(n, Hq * D, device=DEV).bfloat16(), _status()
    runs = torch.tensor([[1, 0, 0, n]], dtype=torch.int32, device=DEV)
    work = torch.zeros(N.shaped_step_work_bytes(2, 1, Hq, Hkv, D, n + 40), dtype=torch.uint8, device=DEV)
    rows, lens = torch.tensor([1, 2], device=DEV).int(), torch.tensor(c.lens, device=DEV).int()
    got = []
    for pdl in (False, True, True):
        shape = dict(Hq=Hq, Hkv=Hkv, D=D, scale=D ** -0.5, status=st, softcap=30.0, slopes=_slopes(Hq), key_pos=c.key_pos, pdl=pdl)
        out, lse, m = torch.zeros_like(q), torch.zeros(n, Hq, device=DEV), torch.zeros(3, Hkv, c.table.shape[1], device=DEV)
        again, step = torch.zeros_like(q), torch.zeros(2, Hq * D, dtype=torch.bfloat16, device=DEV)
        for _ in range(3):
            N.attention_shaped_prompt(q, c.k, c.v, c.table, runs, out, T=n, lse=lse, **shape)
            N.attention_key_mass(q, c.k, c.table, runs, lse, m, T=n, **shape)
            N.attention_shaped_prompt(out, c.k, c.v, c.table, runs, again, T=n, **shape)
            N.attention_shaped_step(again, c.k, c.v, c.table, rows, lens, step, bs=2, E=1, work=work, mass=m, **shape)
        got.append((out, lse, m, again, step))
    torch.cuda.synchronize()
    assert int(st) == 0
    for other in got[1:]:
        assert all(torch.equal(x, y) for x, y in zip(got[0], other))


def test_bad_numbers_on_the_device_raise_the_status_and_read_nothing():
    N = _N()
    c = Cache([100, 100], 2, 64)
    q, out, st = torch.randn(20, 256, device=DEV).bfloat16(), torch.zeros(20, 256, dtype=torch.bfloat16, device=DEV), _status()
    shape = dict(Hq=4, Hkv=2, D=64, scale=0.125, status=st)
    work = torch.zeros(N.shaped_step_work_bytes(2, 1, 4, 2, 64, 200), dtype=torch.uint8, device=DEV)
    want, _, _ = attend(c, [(1, 90, 0, 10)], q, 4, scale=0.125)
    tol = _tolerances(c, q, 4, 0.125, 0.0)[0]
    for bad in ([9, 90, 10, 10], [-1, 90, 10, 10], [2, 200, 10, 10], [2, -5, 10, 10], [2, 90, 15, 10], [2, 90, -1, 10]):
        st.zero_()
        N.attention_shaped_prompt(q, c.k, c.v, c.table, torch.tensor([[1, 90, 0, 10], bad], dtype=torch.int32, device=DEV), out, T=20, **shape)
        assert int(st) == 8 and float((out[:10].double().view(10, 4, 64) - want[:10]).abs().max()) <= tol          # the other sequence is served
    for rows, lens in (([7, 1], [5, 100]), ([1, 2], [100, 400]), ([1, 2], [100, -1])):
        st.zero_()
        N.attention_shaped_step(q, c.k, c.v, c.table, torch.tensor(rows, device=DEV).int(), torch.tensor(lens, device=DEV).int(), out, bs=2, E=1, work=work, **shape)
        assert int(st) == 8
    # pages outside the pool, a row listed twice where weights are added, a workspace too small for the contexts
    table = c.table.clone()
    table[1, 50] = 100000
    table[1, 51] = -3
    m = torch.zeros(3, 2, c.table.shape[1], device=DEV)
    lse = torch.zeros(20, 4, device=DEV)
    for call in (lambda: N.attention_shaped_prompt(q, c.k, c.v, table, torch.tensor([[1, 90, 0, 10]], dtype=torch.int32, device=DEV), out, T=20, **shape),
                 lambda: N.attention_key_mass(q, c.k, table, torch.tensor([[1, 90, 0, 10]], dtype=torch.int32, device=DEV), lse, m, T=20, **shape),
                 lambda: N.attention_key_mass(q, c.k, c.table, torch.tensor([[1, 90, 0, 10], [1, 90, 10, 10]], dtype=torch.int32, device=DEV), lse, m, T=20, **shape),
                 lambda: N.attention_shaped_step(q, c.k, c.v, table, *(torch.tensor(x, device=DEV).int() for x in ([1, 2], [100, 100])), out, bs=2, E=1, work=work, **shape),
                 lambda: N.attention_shaped_step(q, c.k, c.v, c.table, *(torch.tensor(x, device=DEV).int() for x in ([2, 2], [100, 100])), out, bs=2, E=1, work=work, mass=m, **shape),
                 lambda: N.attention_shaped_step(q, c.k, c.v, c.table, *(torch.tensor(x, device=DEV).int() for x in ([1, 2], [100, 100])), out, bs=2, E=1, mass=m,
                                                 work=work[:N.shaped_step_work_bytes(2, 1, 4, 2, 64) + 2 * 128 * 4 * 4], **shape)):
        st.zero_()
        call()
        assert int(st) == 8


def test_arguments_that_do_not_fit_are_refused():
    N = _N()
    c = Cache([20], 2, 64)
    q, st, runs = torch.zeros(20, 256, dtype=torch.bfloat16, device=DEV), _status(), torch.tensor([[1, 0, 0, 20]], dtype=torch.int32, device=DEV)
    good = dict(q=q, k_pool=c.k, v_pool=c.v, block_table=c.table, runs=runs, out=q.clone(), T=20, Hq=4, Hkv=2, D=64, scale=0.125, status=st)
    N.attention_shaped_prompt(**good)
    z = lambda *s, **k: torch.zeros(*s, device=DEV, **k)                                # noqa: E731
    for bad in (dict(q=q.float()), dict(q=q[:10]), dict(q=q[:, :128]), dict(q=q.T), dict(out=q.cpu()), dict(k_pool=c.k.to(torch.uint8)), dict(k_pool=c.k[:, :64]), dict(v_pool=c.v.float()),
                dict(block_table=c.table.long()), dict(runs=runs.long()), dict(runs=runs[0]), dict(slopes=z(3)), dict(slopes=z(4, dtype=torch.float64)), dict(bounds=z(20, 2)),
                dict(bounds=z(19, 2, dtype=torch.int32)), dict(key_pos=c.table[:, :4]), dict(lse=z(19, 4)), dict(lse=z(20, 4, dtype=torch.bfloat16)), dict(status=st.long())):
        with pytest.raises(ValueError):
            N.attention_shaped_prompt(**{**good, **bad})
    m = z(2, 2, c.table.shape[1])
    for bad in (m[:1], m[:, :1], m[:, :, :3], m.double(), m.transpose(1, 2), z(4, 2, c.table.shape[1])[::2]):
        with pytest.raises(ValueError):
            N.attention_key_mass(q, c.k, c.table, runs, z(20, 4), bad, T=20, Hq=4, Hkv=2, D=64, scale=0.125, status=st)


# ------------------------------------------------------------------------------- eviction
def _rows(lens, heads, *, width=None, seed=0, shared=0, ties=False):
    """Rows 1.. with their pages, the first ``shared`` of them held by all; weights, positions and an allocator in which somebody else holds a page too."""
    from smcsd_b200.memory.pools import PageAllocator
    g = torch.Generator(device=DEV).manual_seed(seed)
    a = PageAllocator(sum(lens) + 200, DEV)
    width = width or max(lens) + 4
    table = torch.zeros(2 * len(lens) + 1, width, dtype=torch.int32, device=DEV)
    common = a.alloc(shared)
    for i, n in enumerate(lens):
        s = min(shared, n)
        table[i + 1, :s] = common[:s]
        if n > s:
            table[i + 1, s:n] = a.alloc(n - s)
        a.refcount.index_add_(0, common[:s].long(), torch.ones(s, dtype=torch.int32, device=DEV))
    if shared:
        a.dec_ref_and_free(common)
    mass = torch.rand(table.shape[0], heads, width, device=DEV, generator=g)
    if ties:
        mass = (mass * 3).floor()
    ln = torch.tensor([0] + lens + [0] * len(lens), dtype=torch.int32, device=DEV)
    mass *= torch.arange(width, device=DEV) < ln[:, None, None]
    pos = (torch.arange(width, device=DEV) * 2).int().repeat(table.shape[0], 1)
    return a, table, mass, pos, ln


def _evict(a, table, mass, pos, ln, src, dst, keep, first, last, work=None):
    N = _N()
    st, kept = _status(), torch.full((len(src), keep), -7, dtype=torch.int32, device=DEV)
    work = torch.zeros(N.evict_work_bytes(a.size), dtype=torch.uint8, device=DEV) if work is None else work
    N.evict_tokens(table, *(torch.tensor(x, device=DEV).int() for x in (src, dst)), ln, mass, a.refcount, a.free_stack, a.free_count, keep=keep, first=first, last=last, key_pos=pos,
                   kept=kept, work=work, status=st)
    torch.cuda.synchronize()
    return kept, int(st), work


@pytest.mark.parametrize("heads,lens,shared,keep,first,last,ties", [
    (1, [1, 0, 5], 0, 3, 1, 1, False), (2, [40, 41, 39], 10, 40, 4, 4, True), (8, [1000, 513, 512, 511], 300, 200, 0, 0, True), (3, [1025, 77], 50, 64, 16, 48, False),
    (4, [9000, 20000], 5000, 3000, 4, 100, True), (8, [30000], 0, 1, 0, 1, False), (2, [8192, 8193], 100, 8191, 0, 8191, True), (5, [300] * 20, 128, 130, 2, 5, True)])
def test_evict_in_place_and_into_other_rows(heads, lens, shared, keep, first, last, ties):
    """Pages, positions, weights, lengths, references and the free stack against plain sorting and the allocator's host form."""
    for fork in (False, True):
        a, table, mass, pos, ln = _rows(lens, heads, shared=shared, ties=ties)
        b, t0, m0, p0, l0 = _rows(lens, heads, shared=shared, ties=ties)
        n = len(lens)
        src = list(range(1, n + 1))
        dst = [s + n for s in src] if fork else src
        kept, st, work = _evict(a, table, mass, pos, ln, src, dst, keep, first, last)
        assert st == 0 and not bool(work[:256].any()) and not bool(work[256 + 4 * 4096:].any())          # counters and marks are zero again
        gone = []
        for i, (s, d) in enumerate(zip(src, dst)):
            stay = choose(head_sums(m0[s, :, :lens[i]]).tolist(), keep, first, last) if lens[i] else []
            assert kept[i].tolist() == stay + [-1] * (keep - len(stay))
            at = torch.tensor(stay, dtype=torch.long, device=DEV)
            k = len(stay)
            assert int(ln[d]) == k and torch.equal(table[d, :k], t0[s][at]) and torch.equal(pos[d, :k], p0[s][at]) and torch.equal(mass[d, :, :k], m0[s][:, at])
            assert not bool(mass[d, :, k:].any())
            if fork:
                assert torch.equal(table[s], t0[s]) and torch.equal(mass[s], m0[s]) and int(ln[s]) == lens[i]
                b.inc_ref(t0[s][at])
            else:
                out = torch.ones(lens[i], dtype=torch.bool, device=DEV)
                out[at] = False
                gone.append(t0[s, :lens[i]][out])
        if not fork:
            b.dec_ref_and_free(torch.cat(gone))
        assert torch.equal(a.refcount[1:], b.refcount[1:]) and int(a.free_count) == int(b.free_count)
        assert torch.equal(a.free_stack[:int(a.free_count)], b.free_stack[:int(b.free_count)])
        if not fork:
            a.check_conservation()


def test_evict_orders_nan_infinities_and_zeros():
    a, table, mass, pos, ln = _rows([12], 1)
    mass[1, 0, :12] = torch.tensor([0.0, -0.0, float("nan"), float("inf"), 1.0, -1.0, float("-inf"), 1e-42, 1.0, 2.0, 3.0, 0.0], device=DEV)
    kept, st, _ = _evict(a, table, mass, pos, ln, [1], [2], 8, 0, 0)
    assert st == 0 and kept[0].tolist() == [0, 2, 3, 4, 7, 8, 9, 10]


def test_evict_refuses_rows_that_several_entries_touch():
    """Rows written twice, or written and read: those entries are left alone, the others are served."""
    for src, dst, bad in (([1, 1, 2], [3, 3, 4], {0, 1}), ([1, 2, 3], [1, 1, 6], {0, 1}), ([1, 2], [2, 4], {0, 1}), ([1, 2], [1, 99], {1}), ([-1, 2], [1, 2], {0}), ([1, 2, 1], [4, 4, 5], {0, 1})):
        a, table, mass, pos, ln = _rows([50, 60, 70], 2)
        t0, l0, m0, r0 = table.clone(), ln.clone(), mass.clone(), a.refcount.clone()
        kept, st, _ = _evict(a, table, mass, pos, ln, src, dst, 20, 2, 2)
        assert st == 8
        for i, (s, d) in enumerate(zip(src, dst)):
            if i not in bad:
                stay = choose(head_sums(m0[s, :, :int(l0[s])]).tolist(), 20, 2, 2)
                assert int(ln[d]) == 20 and kept[i].tolist() == stay and torch.equal(table[d, :20], t0[s][torch.tensor(stay, device=DEV)])
            elif 0 <= d < 7:
                assert int(ln[d]) == int(l0[d]) and torch.equal(table[d], t0[d]) and torch.equal(mass[d], m0[d])
        if all(i in bad for i in range(len(src))):
            assert torch.equal(a.refcount, r0)


def test_prompt_mass_eviction_and_steps_together():
    """A prompt with its weights, a row brought to a budget and a fork of it, tokens appended to both, a step that adds to the weights, evicted again: captured whole
    and replayed, against the oracle on what is left of the cache."""
    N = _N()
    Hq, Hkv, D, n, keep, cap = 8, 2, 64, 500, 150, 30.0
    from smcsd_b200.memory.pools import PageAllocator
    c = Cache([n], Hkv, D, order="up", seed=5, spare=40)
    a = PageAllocator(n + 40, DEV)
    pages = a.alloc(n)
    width = n + 8
    table = torch.zeros(3, width, dtype=torch.int32, device=DEV)
    table[1, :n] = pages
    pos = torch.zeros_like(table)
    pos[1, :n] = torch.arange(n, device=DEV)
    ln, st = torch.tensor([0, n, 0], device=DEV).int(), _status()
    mass, slopes = torch.zeros(3, Hkv, width, device=DEV), _slopes(Hq)
    c.table, c.key_pos, c.lens = table, pos, [n, 0]
    q, q1 = torch.randn(n, Hq * D, device=DEV).bfloat16(), torch.randn(2, Hq * D, device=DEV).bfloat16()
    new_k, new_v = (torch.randn(2, Hkv * D, device=DEV).bfloat16() for _ in range(2))
    out, lse, out1 = torch.zeros_like(q), torch.zeros(n, Hq, device=DEV), torch.zeros_like(q1)
    kept, whole, kept2 = (torch.zeros(*x, dtype=torch.int32, device=DEV) for x in ((1, keep), (1, keep), (2, 100)))
    ework = torch.zeros(N.evict_work_bytes(a.size), dtype=torch.uint8, device=DEV)
    swork = torch.zeros(N.shaped_step_work_bytes(2, 1, Hq, Hkv, D, 2 * (keep + 1)), dtype=torch.uint8, device=DEV)
    one, two, both = (torch.tensor(x, device=DEV).int() for x in ([1], [2], [1, 2]))
    fresh, runs = a.alloc(2), torch.tensor([[1, 0, 0, n]], dtype=torch.int32, device=DEV)
    shape = dict(Hq=Hq, Hkv=Hkv, D=D, scale=0.125, status=st, softcap=cap, slopes=slopes, key_pos=pos)
    start = [t.clone() for t in (table, pos, ln, mass, a.refcount, a.free_stack, a.free_count)]

    def chain():
        for t, s in zip((table, pos, ln, mass, a.refcount, a.free_stack, a.free_count), start):
            t.copy_(s)
        N.attention_shaped_prompt(q, c.k, c.v, table, runs, out, T=n, lse=lse, **shape)
        N.attention_key_mass(q, c.k, table, runs, lse, mass, T=n, **shape)
        pool = (a.refcount, a.free_stack, a.free_count)
        N.evict_tokens(table, one, one, ln, mass, *pool, keep=keep, first=4, last=30, key_pos=pos, kept=kept, work=ework, status=st)
        N.evict_tokens(table, one, two, ln, mass, *pool, keep=keep, first=4, last=30, key_pos=pos, kept=whole, work=ework, status=st)        # all that is left of it
        for i in (0, 1):                                             # the next token of either row
            table[i + 1, keep] = fresh[i]
            pos[i + 1, keep].fill_(n)
        c.k.index_copy_(0, fresh.long(), new_k)
        c.v.index_copy_(0, fresh.long(), new_v)
        ln[1:] += 1
        N.attention_shaped_step(q1, c.k, c.v, table, both, ln[1:], out1, bs=2, E=1, work=swork, mass=mass, **shape)
        N.evict_tokens(table, both, both, ln, mass, *pool, keep=100, first=4, last=30, key_pos=pos, kept=kept2, work=ework, status=st)

    chain()
    torch.cuda.synchronize()
    first = [t.clone() for t in (out, out1, table, pos, ln, mass, kept2, a.refcount, a.free_stack)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        chain()
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert int(st) == 0 and all(torch.equal(x, y) for x, y in zip(first, (out, out1, table, pos, ln, mass, kept2, a.refcount, a.free_stack)))

    # the oracle, from the prompt on; the selection follows the weights as the kernels made them (each is held to the oracle's within its tolerance above)
    want, _, w = attend(type("C", (), dict(k=c.k, v=c.v, table=start[0], key_pos=start[1], D=D, Hkv=Hkv, lens=[n, 0], positions=lambda self, r: start[1][r, :n].long()))(),
                        [(1, 0, 0, n)], q, Hq, scale=0.125, softcap=cap, slopes=slopes)
    assert float((out.double().view(want.shape) - want).abs().max()) <= _tolerances(c, q, Hq, 0.125, cap)[0]
    order = w[1].sum(0)[4:n - 30].sort(descending=True).values
    inner = kept[0, 4:keep - 30].long()
    assert float(w[1].sum(0)[inner].min()) >= float(order[keep - 34 - 1]) * (1 - 1e-4)
    at = torch.cat([kept[0].long(), torch.tensor([n], device=DEV)])
    kk, vv = (torch.cat([x[pages.long()][kept[0].long()], y[:1]]) for x, y in ((c.k, new_k), (c.v, new_v)))
    s = torch.einsum("hd,khd->hk", q1[0].view(Hq, D).double(), kk.view(-1, Hkv, D).double().repeat_interleave(Hq // Hkv, 1)) * 0.125
    s = cap * torch.tanh(s / cap) - slopes.double()[:, None] * (n - at)
    o = torch.einsum("hk,khd->hd", s.softmax(-1), vv.view(-1, Hkv, D).double().repeat_interleave(Hq // Hkv, 1))
    assert float((out1[0].double().view(Hq, D) - o).abs().max()) <= _tolerances(c, q1, Hq, 0.125, cap)[0]
    assert ln.tolist() == [0, 100, 100] and int((a.refcount[1:] > 0).sum()) + int(a.free_count) == a.size
