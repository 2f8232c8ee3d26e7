"""Shaped attention where caches, masks and numbers are at their edges, on the GPU against float64 (shaped_oracle.py)."""
import math

import pytest
import torch

from shaped_oracle import Cache, attend

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _N():
    from smcsd_b200.ops import native_shaped as N
    return N


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _slopes(Hq):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], device=DEV)


def _randn(*shape, seed=0):
    """bf16 from a generator of its own: the default one's order belongs to the other tests."""
    return torch.randn(*shape, device=DEV, generator=torch.Generator(DEV).manual_seed(seed)).bfloat16()


def _out_error(c, moved):
    """An output's: every probability and the output itself are rounded to bf16, by 2^-8 of themselves at most (half a step), and a score's error moves a probability by as much,
    against the sum of all once more."""
    return (2 * 2.0 ** -8 + 2 * moved) * float(c.v[1:].double().abs().max())


def _score_error(c, q, scale):
    """How far a score may be off: products of D values summed in fp32, every addition by at most 2^-23 of the largest partial sum, |q||k| scale."""
    big = float((q.double().view(-1, c.D).norm(dim=1).max() * c.k[1:].double().view(-1, c.D).norm(dim=1).max()) * scale)
    return c.D / 16 * 2.0 ** -23 * big


# ------------------------------------------------------------------------------- gaps in the positions
def _gap_cache(lens, Hkv, D, ahead, gap, seed):
    """Rows of which ``ahead`` tokens lie at the front, the others ``gap`` positions further on."""
    c = Cache(lens, Hkv, D, seed=seed, order="up", shed=True)
    at = torch.arange(c.table.shape[1], device=DEV)
    c.key_pos[:] = at + gap * (at >= ahead)
    return c


@pytest.mark.parametrize("gap", [6 * 10 ** 4, 10 ** 6, 2 ** 24 - 2000])
@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 64), (16, 4, 128), (16, 2, 256)])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_distance_bias_across_a_gap_inside_a_step(gap, Hq, Hkv, D, softcap):
    """Held tokens fill whole steps of keys, of which the first ones lie far in front of the rest: the distances of the near ones must not drown in those.  A weight is off by
    what the score is, the log-sum-exp by that and half a unit in the last place of an fp32 number of its size (2^-20 covers numbers up to 16)."""
    N = _N()
    held, n = 512, 40
    for ahead in (8, 500):
        c = _gap_cache([held + n, held], Hkv, D, ahead, gap, seed=gap % 97 + ahead)
        runs = [(1, held, 0, n)]
        q, st = _randn(n, Hq * D, seed=gap + D), _int([0])
        kw = dict(scale=D ** -0.5, softcap=softcap, slopes=_slopes(Hq))
        want, want_lse, mass = attend(c, runs, q, Hq, **kw)
        out, lse, m = torch.zeros_like(q), torch.zeros(n, Hq, device=DEV), torch.zeros(3, Hkv, c.table.shape[1], device=DEV)
        kw.update(T=n, Hq=Hq, Hkv=Hkv, D=D, status=st, key_pos=c.key_pos)
        N.attention_shaped_prompt(q, c.k, c.v, c.table, _int(runs), out, lse=lse, **kw)
        N.attention_key_mass(q, c.k, c.table, _int(runs), want_lse.float(), m, **kw)
        torch.cuda.synchronize()
        assert int(st) == 0
        moved = _score_error(c, q, D ** -0.5) + 3e-6 * (softcap or 0.0) + 2.0 ** -20
        assert float((lse.double() - want_lse).abs().max()) <= moved
        assert float((out.double().view(want.shape) - want).abs().max()) <= _out_error(c, moved)
        w = mass[1]
        # weights far below a key's sum may be rounded away: the bias of a far key is as large as its distance, and so is its rounding, but exp of it is nothing
        assert bool(((m[1, :, :w.shape[1]].double() - w).abs() <= 2 * moved * w + 1e-12).all())


@pytest.mark.parametrize("slope", [-0.002, -0.3])
def test_distance_bias_that_grows_across_a_gap(slope):
    """A negative slope favours the far tokens: those at the other end of the step have to be right then.  Scores grow with the distance and so does what fp32 can tell of
    them: half a unit of the largest, once for the product and once for the sum, in the score and in the reference."""
    N = _N()
    held, n, Hq, D, gap = 256, 30, 4, 64, 5000
    c = _gap_cache([held + n], 1, D, 100, gap, seed=3)
    runs, slopes = [(1, held, 0, n)], torch.full((Hq,), slope, device=DEV)
    q, st = _randn(n, Hq * D, seed=gap + D), _int([0])
    want, want_lse, mass = attend(c, runs, q, Hq, scale=0.125, slopes=slopes)
    out, lse, m = torch.zeros_like(q), torch.zeros(n, Hq, device=DEV), torch.zeros(2, 1, c.table.shape[1], device=DEV)
    kw = dict(scale=0.125, slopes=slopes, T=n, Hq=Hq, Hkv=1, D=D, status=st, key_pos=c.key_pos)
    N.attention_shaped_prompt(q, c.k, c.v, c.table, _int(runs), out, lse=lse, **kw)
    N.attention_key_mass(q, c.k, c.table, _int(runs), lse, m, **kw)
    torch.cuda.synchronize()
    moved = _score_error(c, q, 0.125) + 4 * 2.0 ** -24 * -slope * (gap + held + n) * 1.5 + 2.0 ** -20
    assert int(st) == 0 and float((lse.double() - want_lse).abs().max()) <= moved
    assert float((out.double().view(want.shape) - want).abs().max()) <= _out_error(c, moved)
    w = mass[1]
    assert bool(((m[1, :, :w.shape[1]].double() - w).abs() <= 2 * moved * w + 1e-12).all())


# ------------------------------------------------------------------------------- caps far below and above the scores
@pytest.mark.parametrize("cap", [1e-30, 1e-8, 1e-6, 1e-3, 1e5, 1e30])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (8, 2, 128), (8, 2, 256)])
def test_caps_far_from_the_scores(cap, Hq, Hkv, D):
    """Scores of zero too: a key tile, a row of tokens and a whole sequence of them beside ordinary ones.  A capped score is off by 3e-6 of itself, an uncapped one by its
    product's error."""
    N = _N()
    c = Cache([300, 150], Hkv, D, seed=2)
    q, st = _randn(450, Hq * D, seed=8), _int([0])
    q[40:170] = 0
    q[300:] = 0
    c.k[c.table[1, 128:256].long()] = 0
    runs, scale = [(1, 0, 0, 300), (2, 0, 300, 150)], D ** -0.5
    want, want_lse, mass = attend(c, runs, q, Hq, scale=scale, softcap=cap)
    out, lse, m = torch.zeros_like(q), torch.zeros(450, Hq, device=DEV), torch.zeros(3, Hkv, c.table.shape[1], device=DEV)
    kw = dict(Hq=Hq, Hkv=Hkv, D=D, scale=scale, softcap=cap, status=st)
    N.attention_shaped_prompt(q, c.k, c.v, c.table, _int(runs), out, T=450, lse=lse, **kw)
    N.attention_key_mass(q, c.k, c.table, _int(runs), lse, m, T=450, **kw)
    work = torch.zeros(N.shaped_step_work_bytes(2, 1, Hq, Hkv, D), dtype=torch.uint8, device=DEV)
    out1, lse1 = torch.zeros(2, Hq * D, dtype=torch.bfloat16, device=DEV), torch.zeros(2, Hq, device=DEV)
    N.attention_shaped_step(q[[299, 449]], c.k, c.v, c.table, _int([1, 2]), _int([300, 150]), out1, bs=2, E=1, work=work, lse=lse1, **kw)
    torch.cuda.synchronize()
    assert int(st) == 0
    moved = _score_error(c, q, scale) + 3e-6 * min(cap, 30.0) + 2.0 ** -20
    for o, l, at in ((out, lse, slice(None)), (out1, lse1, [299, 449])):
        assert float((o.double().view(-1, Hq, D) - want[at]).abs().max()) <= _out_error(c, moved)
        assert float((l.double() - want_lse[at]).abs().max()) <= moved
    for row, w in mass.items():
        assert bool(((m[row, :, :w.shape[1]].double() - w).abs() <= 2 * moved * w + 1e-12).all())


# ------------------------------------------------------------------------------- a workspace that contexts have outgrown
def test_step_behind_one_whose_workspace_was_too_small():
    """The refused weights raise the status; the step's outputs are there for whoever comes next, also for one that starts early, and the workspace is fit for the next step."""
    N = _N()
    Hq, Hkv, D = 8, 2, 64
    c = Cache([9000, 8000], Hkv, D, seed=4)
    q, st = _randn(2, Hq * D, seed=5), _int([0])
    rows, lens = _int([1, 2]), _int(c.lens)
    want, _, mass = attend(c, [(1, 8999, 0, 1), (2, 7999, 1, 1)], q, Hq, scale=0.125)
    tol = _out_error(c, _score_error(c, q, 0.125) + 2.0 ** -20)
    small = N.shaped_step_work_bytes(2, 1, Hq, Hkv, D, 300)
    work = torch.zeros(N.shaped_step_work_bytes(2, 1, Hq, Hkv, D, 17000), dtype=torch.uint8, device=DEV)
    outs = [torch.zeros_like(q) for _ in range(8)]
    m = [torch.zeros(3, Hkv, c.table.shape[1], device=DEV) for _ in range(2)]
    kw = dict(bs=2, E=1, Hq=Hq, Hkv=Hkv, D=D, scale=0.125, status=st)

    def chain():
        for i in range(0, 8, 2):
            N.attention_shaped_step(q, c.k, c.v, c.table, rows, lens, outs[i], work=work[:small], mass=m[0], **kw)
            N.attention_shaped_step(outs[i], c.k, c.v, c.table, rows, lens, outs[i + 1], work=work, pdl=True, **kw)
    chain()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        chain()
    g.replay()
    torch.cuda.synchronize()
    assert int(st) == 8 and not bool(m[0].any())
    again, _, _ = attend(c, [(1, 8999, 0, 1), (2, 7999, 1, 1)], outs[0], Hq, scale=0.125)
    for i in range(0, 8, 2):
        assert torch.equal(outs[i], outs[0]) and torch.equal(outs[i + 1], outs[1])
    assert float((outs[0].double().view(want.shape) - want).abs().max()) <= tol
    assert float((outs[1].double().view(want.shape) - again).abs().max()) <= tol
    st.zero_()
    N.attention_shaped_step(q, c.k, c.v, c.table, rows, lens, outs[0], work=work, mass=m[1], **kw)
    torch.cuda.synchronize()
    assert int(st) == 0 and torch.equal(outs[0], outs[2])
    for row, w in mass.items():
        moved = _score_error(c, q, 0.125) + 2.0 ** -20
        assert bool(((m[1][row, :, :w.shape[1]].double() - w).abs() <= 2 * moved * w + 1e-12).all())


# ------------------------------------------------------------------------------- listed positions
@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 64), (16, 4, 128), (16, 2, 256)])
def test_listed_positions_are_there_when_their_keys_are(Hq, Hkv, D):
    """A hundred replays of a step whose masks and distances rest on listed positions, caches and positions changing place between them: the same bits as at first."""
    N = _N()
    lens = [2500, 700, 64, 3000]
    c = Cache(lens, Hkv, D, seed=6, shed=True)
    q, st = _randn(4, Hq * D, seed=7), _int([0])
    work = torch.zeros(N.shaped_step_work_bytes(4, 1, Hq, Hkv, D), dtype=torch.uint8, device=DEV)
    own = torch.stack([c.key_pos[i + 1, n - 1] for i, n in enumerate(lens)])
    bounds, slopes, scale = N.score_bounds(own, window=900), _slopes(Hq), D ** -0.5
    want, _, _ = attend(c, [(i + 1, n - 1, i, 1) for i, n in enumerate(lens)], q, Hq, scale=scale, slopes=slopes, bounds=bounds)
    out, other = torch.zeros_like(q), torch.zeros_like(q)
    kw = dict(bs=4, E=1, Hq=Hq, Hkv=Hkv, D=D, scale=scale, status=st, work=work, slopes=slopes)
    g = torch.cuda.CUDAGraph()
    far = c.key_pos + 5

    def step(o, pos):
        N.attention_shaped_step(q, c.k, c.v, c.table, _rows, _lens, o, bounds=bounds if pos is c.key_pos else shifted, key_pos=pos, **kw)
    _rows, _lens, shifted = _int([1, 2, 3, 4]), _int(lens), bounds + 5
    step(out, c.key_pos)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        step(other, far)                                             # the same distances and masks
        step(out, c.key_pos)
    first = out.clone()
    assert float((first.double().view(want.shape) - want).abs().max()) <= _out_error(c, _score_error(c, q, scale) + 2.0 ** -20)
    for _ in range(100):
        g.replay()
        assert torch.equal(out, first)
    assert torch.equal(other, first) and int(st) == 0


# ------------------------------------------------------------------------------- tables that are columns of wider ones
def _allocator(pages):
    """Every page held once; free stack and its count."""
    return torch.ones(pages + 1, dtype=torch.int32, device=DEV), torch.zeros(pages, dtype=torch.int32, device=DEV), _int([0])


def test_columns_of_a_wider_table():
    """Positions and weights of as many columns as the slice: the same results as with tensors of their own, and lengths that reach into the other columns raise the status."""
    N = _N()
    Hq, Hkv, D, cols = 8, 2, 64, 210
    c = Cache([200, 150], Hkv, D, seed=12, shed=True)
    wide = torch.full((3, 400), 1, dtype=torch.int32, device=DEV)
    wide[:, :205] = c.table
    pos = torch.zeros(3, cols, dtype=torch.int32, device=DEV)
    pos[:, :205] = c.key_pos
    own = wide[:, :cols].contiguous()
    q, results = _randn(60, Hq * D, seed=13), []
    work = torch.zeros(N.shaped_step_work_bytes(2, 1, Hq, Hkv, D, 700), dtype=torch.uint8, device=DEV)
    ework = torch.zeros(N.evict_work_bytes(350), dtype=torch.uint8, device=DEV)

    def run(table, held, n0, lens):
        st = _int([0])
        m = torch.zeros(3, Hkv, cols, device=DEV)
        out, lse, out1 = torch.zeros_like(q), torch.zeros(60, Hq, device=DEV), torch.zeros(2, Hq * D, dtype=torch.bfloat16, device=DEV)
        kw = dict(Hq=Hq, Hkv=Hkv, D=D, scale=0.125, status=st, key_pos=pos, slopes=_slopes(Hq))
        runs = _int([[1, held, 0, n0], [2, 130, 40, 20]])
        states = []
        N.attention_shaped_prompt(q, c.k, c.v, table, runs, out, T=60, lse=lse, **kw)
        states.append(int(st.clone()))
        st.zero_()
        N.attention_key_mass(q, c.k, table, runs, lse, m, T=60, **kw)
        states.append(int(st.clone()))
        st.zero_()
        N.attention_shaped_step(q[:2], c.k, c.v, table, _int([1, 2]), _int(lens), out1, bs=2, E=1, work=work, mass=m, **kw)
        states.append(int(st.clone()))
        st.zero_()
        t, p, ln = (table if table.is_contiguous() else wide.clone()[:, :cols]), pos.clone(), _int([0] + lens)
        t = t.clone() if table.is_contiguous() else t
        kept, mass = torch.full((2, 90), -7, dtype=torch.int32, device=DEV), m.clone()
        refs, stack, count = _allocator(350)
        N.evict_tokens(t, _int([1, 2]), _int([1, 2]), ln, mass, refs, stack, count, keep=90, first=2, last=9, kept=kept, work=ework, status=st, key_pos=p)
        states.append(int(st.clone()))
        return states, [out, lse, out1, m, t.clone(), p, ln, kept, mass, refs, stack, count]

    for table in (own, wide[:, :cols]):
        states, got = run(table, 160, 40, [200, 150])
        assert states == [0, 0, 0, 0]
        results.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*results))
    # beyond the columns, within the pitch: that sequence is refused, the other one served
    states, bad = run(wide[:, :cols], 180, 40, [215, 150])
    assert states == [8, 8, 8, 8]
    assert not bool(bad[0][:40].any()) and not bool(bad[2][0].any()) and torch.equal(bad[0][40:], results[0][0][40:]) and torch.equal(bad[2][1], results[0][2][1])
    assert not bool(bad[3][1].any()) and bad[6].tolist() == [0, 215, 90]


# ------------------------------------------------------------------------------- what no token sees
@pytest.mark.parametrize("Hq,Hkv,D,E", [(32, 8, 64, 1), (16, 4, 128, 1), (16, 4, 128, 5), (16, 2, 256, 1), (16, 2, 256, 2)])
@pytest.mark.parametrize("shed", [False, True])
@pytest.mark.parametrize("copies", [1, 6, 12])
def test_step_reads_nothing_outside_of_the_intervals(Hq, Hkv, D, E, shed, copies):
    """Keys and values that no token of their sequence sees are NaN: a window's, a document's, those ahead of where a mask ends, all of a sequence whose masks are empty."""
    N = _N()
    lens = [900, 300, 64, 1, 2000, 517, 130] * copies
    bs = len(lens)
    c = Cache(lens, Hkv, D, seed=D + E, shed=shed)
    runs = [(i + 1, n - E, i * E, E) for i, n in enumerate(lens)]
    b = torch.zeros(bs * E, 2, dtype=torch.int32, device=DEV)
    for i, n in enumerate(lens):
        pos = c.positions(i + 1)
        own = torch.cat([torch.full((max(0, E - n),), -1, device=DEV), pos[max(n - E, 0):]])
        last = int(pos[-1])
        b[i * E:(i + 1) * E] = (N.score_bounds(own, window=100), N.score_bounds(own, doc_first=own.clamp(min=0) // 290 * 290), _int([[last // 4, last // 2]] * E),
                                N.score_bounds(own), _int([[9, 8]] * E), _int([[0, last // 3]] * E), _int([[last + 1, last + 50]] * E))[i % 7]
        see = b[i * E + max(0, E - n):(i + 1) * E]
        see = see[see[:, 0] <= see[:, 1]]
        unseen = (pos < see[:, 0].min()) | (pos > see[:, 1].max()) if len(see) else torch.ones_like(pos, dtype=torch.bool)
        hidden = c.table[i + 1, :n][unseen].long()
        c.k[hidden] = c.v[hidden] = float("nan")
    q, st = _randn(bs * E, Hq * D, seed=14), _int([0])
    clean = Cache(lens, Hkv, D, seed=D + E, shed=shed)
    want, want_lse, mass = attend(clean, runs, q, Hq, scale=D ** -0.5, softcap=20.0, bounds=b)
    out, lse, m = torch.zeros_like(q), torch.zeros(bs * E, Hq, device=DEV), torch.zeros(bs + 1, Hkv, c.table.shape[1], device=DEV)
    work = torch.zeros(N.shaped_step_work_bytes(bs, E, Hq, Hkv, D, sum(lens)), dtype=torch.uint8, device=DEV)
    N.attention_shaped_step(q, c.k, c.v, c.table, torch.arange(1, bs + 1, device=DEV).int(), _int(lens), out, bs=bs, E=E, Hq=Hq, Hkv=Hkv, D=D, scale=D ** -0.5, softcap=20.0,
                            status=st, work=work, bounds=b, key_pos=c.key_pos, lse=lse, mass=m)
    torch.cuda.synchronize()
    assert int(st) == 0
    moved = _score_error(clean, q, D ** -0.5) + 3e-6 * 20 + 2.0 ** -20
    assert float((out.double().view(want.shape) - want).abs().max()) <= _out_error(clean, moved)
    there = torch.isfinite(want_lse)
    assert torch.equal(torch.isfinite(lse), there) and float((lse.double() - want_lse)[there].abs().max()) <= moved
    for row, w in mass.items():
        assert bool(((m[row, :, :w.shape[1]].double() - w).abs() <= 2 * moved * w + 1e-12).all())


# ------------------------------------------------------------------------------- the mass of some tokens of a pass
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (16, 4, 128), (6, 2, 128), (8, 1, 256)])
def test_key_mass_bits_depend_on_the_sequence_alone(Hq, Hkv, D):
    """A long sequence alone, beside many short ones, and as some runs of a longer pass: the same bits."""
    N = _N()
    n, got, st = 2100, [], _int([0])
    for others in (0, 40):
        c = Cache([n] + [3] * others, Hkv, D, seed=21, order="up")
        c.k[1:n + 1] = _randn(n, Hkv * D, seed=22)
        q = torch.cat([_randn(n, Hq * D, seed=23), _randn(3 * others, Hq * D, seed=24)])
        lse = torch.full((len(q), Hq), 4.0, device=DEV)
        runs = [[1, 0, 0, n]] + [[2 + i, 0, n + 3 * i, 3] for i in range(others)]
        kw = dict(Hq=Hq, Hkv=Hkv, D=D, scale=D ** -0.5, status=st, softcap=30.0)
        for listed in (runs, runs[:1], runs[::-1]):
            m = torch.zeros(others + 2, Hkv, c.table.shape[1], device=DEV)
            N.attention_key_mass(q, c.k, c.table, _int(listed), lse, m, T=len(q), **kw)
            got.append(m[1, :, :n].clone())
    torch.cuda.synchronize()
    assert int(st) == 0 and all(torch.equal(got[0], x) for x in got[1:])


@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 64), (16, 4, 128), (16, 2, 256)])
@pytest.mark.parametrize("mask", ["causal", "window", "prefix"])
def test_key_mass_of_the_last_tokens_of_a_pass(Hq, Hkv, D, mask):
    """``runs`` lists the last tokens of each prompt of a pass: their mass alone, and the bits of a call that is handed those tokens only."""
    N = _N()
    sizes, tail = [3000, 40, 900], [64, 40, 33]
    c = Cache(sizes, Hkv, D, seed=25, shed=True)
    T, starts = sum(sizes), [0, 3000, 3040]
    q, st, scale = _randn(T, Hq * D, seed=26), _int([0]), D ** -0.5
    pos = torch.cat([c.positions(i + 1) for i in range(3)])
    b = {"causal": None, "window": N.score_bounds(pos, window=500), "prefix": N.score_bounds(pos, prefix=300)}[mask]
    tails = [(i + 1, n - k, at + n - k, k) for i, (n, k, at) in enumerate(zip(sizes, tail, starts))]
    kw = dict(Hq=Hq, Hkv=Hkv, D=D, scale=scale, status=st, key_pos=c.key_pos, softcap=30.0, slopes=_slopes(Hq))
    _, want_lse, mass = attend(c, tails, q, Hq, scale=scale, softcap=30.0, slopes=_slopes(Hq), bounds=b)
    lse = want_lse.float()
    m = [torch.zeros(4, Hkv, c.table.shape[1], device=DEV) for _ in range(2)]
    N.attention_key_mass(q, c.k, c.table, _int(tails), lse, m[0], T=T, bounds=b, **kw)
    take = torch.cat([torch.arange(at, at + k, device=DEV) for _, _, at, k in tails])
    alone, at = [], 0
    for row, held, _, k in tails:
        alone.append((row, held, at, k))
        at += k
    N.attention_key_mass(q[take], c.k, c.table, _int(alone), lse[take], m[1], T=len(take), bounds=None if b is None else b[take].contiguous(), **kw)
    torch.cuda.synchronize()
    assert int(st) == 0 and torch.equal(m[0], m[1])
    moved = _score_error(c, q, scale) + 3e-6 * 30 + 2.0 ** -20
    for row, w in mass.items():
        assert bool(((m[0][row, :, :w.shape[1]].double() - w).abs() <= 2 * moved * w + 1e-12).all())


# ------------------------------------------------------------------------------- eviction
def test_evict_from_a_table_of_more_columns_than_it_takes():
    """Refused by name; a slice of the table is served, and rows of 262,144 tokens are."""
    N = _N()
    n, width, st = 262144, 300000, _int([0])
    wide = torch.arange(1, width + 1, dtype=torch.int32, device=DEV).repeat(2, 1)
    mass = torch.rand(2, 1, width, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    refs, stack, count = _allocator(width)
    work = torch.zeros(N.evict_work_bytes(width), dtype=torch.uint8, device=DEV)
    lens, kept, one = _int([0, n]), torch.zeros(1, 100, dtype=torch.int32, device=DEV), _int([1])
    args = dict(keep=100, first=4, last=10, kept=kept, work=work, status=st)
    with pytest.raises(ValueError, match="262144"):
        N.evict_tokens(wide, one, one, lens, mass, refs, stack, count, **args)
    with pytest.raises(ValueError, match="4096"):
        N.evict_tokens(wide[:, :n], one.repeat(4097), one.repeat(4097), lens, mass, refs, stack, count, **{**args, "kept": kept.repeat(4097, 1)})
    before = mass[1, 0].clone()
    N.evict_tokens(wide[:, :n], one, one, lens, mass, refs, stack, count, **args)
    torch.cuda.synchronize()
    inner = before[4:n - 10].sort(descending=True, stable=True).indices[:86].sort().values + 4
    want = torch.cat([torch.arange(4, device=DEV), inner, torch.arange(n - 10, n, device=DEV)])
    assert int(st) == 0 and lens.tolist() == [0, 100] and int(count) == n - 100
    assert torch.equal(kept[0].long(), want) and torch.equal(wide[1, :100].long(), want + 1) and torch.equal(mass[1, 0, :100], before[want])
    assert not bool(mass[1, 0, 100:n].any()) and torch.equal(mass[1, 0, n:], before[n:])


def test_evict_with_a_free_count_that_leaves_the_stack():
    """A count below zero or above the pages: the status, and nothing written outside of the stack."""
    N = _N()
    for bad in (-3, 47, 60):
        table = torch.arange(1, 51, dtype=torch.int32, device=DEV).repeat(2, 1)
        mass, lens, st = torch.rand(2, 1, 50, device=DEV, generator=torch.Generator(DEV).manual_seed(2)), _int([0, 50]), _int([0])
        refs = torch.ones(51, dtype=torch.int32, device=DEV)
        stack, count, work = torch.full((150,), -9, dtype=torch.int32, device=DEV), _int([bad]), torch.zeros(N.evict_work_bytes(50), dtype=torch.uint8, device=DEV)
        N.evict_tokens(table, _int([1]), _int([1]), lens, mass, refs, stack[50:100], count, keep=30, first=0, last=0, kept=torch.zeros(1, 30, dtype=torch.int32, device=DEV), work=work,
                       status=st)
        torch.cuda.synchronize()
        assert int(st) == 8 and bool((stack[:50] == -9).all()) and bool((stack[100:] == -9).all()) and int(count) <= 50
        assert not bool(work[:256].any()) and not bool(work[256 + 4 * 4096:].any())


def test_arguments_without_a_page_are_refused():
    N = _N()
    c = Cache([20], 2, 64)
    q, runs = torch.zeros(20, 256, dtype=torch.bfloat16, device=DEV), _int([[1, 0, 0, 20]])
    with pytest.raises(ValueError, match="k_pool"):
        N.attention_shaped_prompt(q, c.k[:0], c.v, c.table, runs, q.clone(), T=20, Hq=4, Hkv=2, D=64, scale=0.125, status=_int([0]))


# ------------------------------------------------------------------------------- runs that share tokens
def test_more_tiles_than_the_queries_have_raise_the_status():
    """Tokens of ``q`` in several runs make more tiles than are launched: some would be left out without a word.  Runs that fill the queries exactly are fine."""
    N = _N()
    c = Cache([100] * 5, 2, 64, seed=30)
    q = _randn(100, 8 * 64, seed=31)
    for runs, want in (([[i + 1, 0, 0, 100] for i in range(5)], 8), ([[1, 0, 0, 65], [2, 0, 65, 1], [3, 0, 66, 1], [4, 0, 67, 1], [5, 0, 68, 32]], 0)):
        st = _int([0])
        N.attention_shaped_prompt(q, c.k, c.v, c.table, _int(runs), torch.zeros_like(q), T=100, Hq=8, Hkv=2, D=64, scale=0.125, status=st)
        assert int(st) == want


# ------------------------------------------------------------------------------- 32-bit results
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (8, 2, 128), (8, 1, 256)])
@pytest.mark.parametrize("softcap", [0.0, 50.0])
@pytest.mark.parametrize("alibi", [False, True])
def test_weights_and_log_sums_keep_their_32_bits(Hq, Hkv, D, softcap, alibi):
    """Root mean squares, beside the worst cases of the other tests.  A score is summed in D / 16 additions, each off by at most 2^-23 of the sum so far, itself no more than a few
    scores; its tanh is off by 6.1e-8 (a log-sum-exp of a prompt's by 3.0e-6 up to 0.35 of the cap and 6.3e-7 beyond), an exponential by 2^-22, a log-sum-exp by 2^-24 of itself."""
    N = _N()
    n, scale = 700, D ** -0.5
    c = Cache([n], Hkv, D, seed=41)
    q, st = (1.6 * _randn(n, Hq * D, seed=42).float()).bfloat16(), _int([0])
    kw = dict(scale=scale, softcap=softcap, slopes=_slopes(Hq) if alibi else None)
    _, want_lse, mass = attend(c, [(1, 0, 0, n)], q, Hq, **kw)
    out, lse, m = torch.zeros_like(q), torch.zeros(n, Hq, device=DEV), torch.zeros(2, Hkv, c.table.shape[1], device=DEV)
    kw.update(T=n, Hq=Hq, Hkv=Hkv, D=D, status=st)
    N.attention_shaped_prompt(q, c.k, c.v, c.table, _int([[1, 0, 0, n]]), out, lse=lse, **kw)
    N.attention_key_mass(q, c.k, c.table, _int([[1, 0, 0, n]]), want_lse.float(), m, **kw)
    torch.cuda.synchronize()
    score = 1.6                                                      # root mean square of q.k scale, for keys of unit variance
    moved = D / 16 * 2.0 ** -23 * 2 * score + 2.0 ** -22 + 2.0 ** -24 * float(want_lse.abs().max())
    off = (m[1, :, :n].double() - mass[1]) / mass[1]
    assert int(st) == 0 and float(off.pow(2).mean().sqrt()) <= moved + (6.1e-8 * 4 * score if softcap else 0.0)
    diff = lse.double() - want_lse
    tanh = max(3.0e-6 * 0.35, 6.3e-7 * 0.75) * softcap
    assert float(diff.pow(2).mean().sqrt()) <= moved + tanh / 2 and float(diff.abs().max()) <= 8 * moved + tanh


def test_rows_of_more_tokens_than_positions_raise_the_status():
    N = _N()
    n = 2 ** 24
    table = torch.ones(1, n + 8, dtype=torch.int32, device=DEV)
    pool, q = torch.ones(2, 64, dtype=torch.bfloat16, device=DEV), torch.ones(1, 64, dtype=torch.bfloat16, device=DEV)
    work = torch.zeros(N.shaped_step_work_bytes(1, 1, 1, 1, 64), dtype=torch.uint8, device=DEV)
    kw = dict(Hq=1, Hkv=1, D=64, scale=0.125)
    for keys, want in ((n, 0), (n + 1, 8)):
        last = _int([[keys - 200, keys - 1]])
        for call in (lambda st, o: N.attention_shaped_prompt(q, pool, pool, table, _int([[0, keys - 1, 0, 1]]), o, T=1, status=st, bounds=last, **kw),
                     lambda st, o: N.attention_shaped_step(q, pool, pool, table, _int([0]), _int([keys]), o, bs=1, E=1, work=work, status=st, bounds=last, **kw)):
            st, out = _int([0]), torch.zeros_like(q)
            call(st, out)
            assert int(st) == want and bool((out == (0.0 if want else 1.0)).all())


@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 64), (16, 4, 128), (16, 2, 256)])
def test_distance_bias_across_a_gap_ahead_of_the_tokens(Hq, Hkv, D):
    """Tokens that see all others, of which many lie behind a gap: the first key of a step is the nearest one then."""
    N = _N()
    n, gap = 600, 10 ** 6
    for ahead in (130, 390):
        c = _gap_cache([n], Hkv, D, ahead, gap, seed=ahead)
        q, st = _randn(n, Hq * D, seed=D), _int([0])
        bounds = _int([[0, 2 ** 24 - 1]] * n)
        kw = dict(scale=D ** -0.5, slopes=_slopes(Hq), bounds=bounds)
        want, want_lse, mass = attend(c, [(1, 0, 0, n)], q, Hq, **kw)
        out, lse, m = torch.zeros_like(q), torch.zeros(n, Hq, device=DEV), torch.zeros(2, Hkv, c.table.shape[1], device=DEV)
        kw.update(T=n, Hq=Hq, Hkv=Hkv, D=D, status=st, key_pos=c.key_pos)
        N.attention_shaped_prompt(q, c.k, c.v, c.table, _int([[1, 0, 0, n]]), out, lse=lse, **kw)
        N.attention_key_mass(q, c.k, c.table, _int([[1, 0, 0, n]]), want_lse.float(), m, **kw)
        torch.cuda.synchronize()
        moved = _score_error(c, q, D ** -0.5) + 2.0 ** -20
        assert int(st) == 0 and float((lse.double() - want_lse).abs().max()) <= moved
        assert float((out.double().view(want.shape) - want).abs().max()) <= _out_error(c, moved)
        assert bool(((m[1, :, :n].double() - mass[1]).abs() <= 2 * moved * mass[1] + 1e-12).all())


@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 64), (16, 4, 128), (16, 2, 256)])
@pytest.mark.parametrize("shed", [False, True])
@pytest.mark.parametrize("softcap,alibi", [(0.0, False), (20.0, True)])
def test_prompts_take_nothing_from_outside_of_the_intervals(Hq, Hkv, D, shed, softcap, alibi):
    """Keys and values that no token of their sequence sees are NaN, ahead of a window, behind where the masks end, and in a sequence whose masks are all empty."""
    N = _N()
    sizes = [(900, 50), (300, 200), (400, 30), (64, 40)]
    c, clean = (Cache([a + n for a, n in sizes], Hkv, D, seed=D, shed=shed) for _ in range(2))
    runs, b, at = [], [], 0
    for i, (held, n) in enumerate(sizes):
        pos = c.positions(i + 1)
        own, last = pos[held:], int(pos[-1])
        see = (N.score_bounds(own, window=100), _int([[last // 4, last // 2]] * n), N.score_bounds(own, doc_first=torch.full_like(own, int(pos[min(200, len(pos) - 1)]))), _int([[9, 8]] * n))[i]
        some = see[see[:, 0] <= see[:, 1]]
        unseen = (pos < some[:, 0].min()) | (pos > some[:, 1].max()) if len(some) else torch.ones_like(pos, dtype=torch.bool)
        hidden = c.table[i + 1, :held + n][unseen].long()
        c.k[hidden] = c.v[hidden] = float("nan")
        runs.append((i + 1, held, at, n))
        b.append(see)
        at += n
    b, q, st, scale = torch.cat(b).contiguous(), _randn(at, Hq * D, seed=3), _int([0]), D ** -0.5
    kw = dict(scale=scale, softcap=softcap, slopes=_slopes(Hq) if alibi else None, bounds=b)
    want, want_lse, mass = attend(clean, runs, q, Hq, **kw)
    out, lse, m = torch.full_like(q, 7.0), torch.zeros(at, Hq, device=DEV), torch.zeros(5, Hkv, c.table.shape[1], device=DEV)
    kw.update(T=at, Hq=Hq, Hkv=Hkv, D=D, status=st, key_pos=c.key_pos)
    N.attention_shaped_prompt(q, c.k, c.v, c.table, _int(runs), out, lse=lse, **kw)
    N.attention_key_mass(q, c.k, c.table, _int(runs), lse, m, **kw)
    torch.cuda.synchronize()
    moved = _score_error(clean, q, scale) + 3e-6 * softcap + 2.0 ** -20
    there = torch.isfinite(want_lse)
    assert int(st) == 0 and float((out.double().view(want.shape) - want).abs().max()) <= _out_error(clean, moved)
    assert torch.equal(torch.isfinite(lse), there) and float((lse.double() - want_lse)[there].abs().max()) <= moved
    for row, w in mass.items():
        assert bool(((m[row, :, :w.shape[1]].double() - w).abs() <= 2 * moved * w + 1e-12).all())
