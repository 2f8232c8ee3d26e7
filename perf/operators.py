"""What the speed of the shaped attention, the key mass and the eviction from the paged cache is measured on.

Attention over a paged cache of one-token pages whose scores are capped by a tanh, lowered by the distance of the tokens, or masked
to an interval of positions per token (causal, a window, documents behind one another, a prefix that all see): ``prompt`` for
many tokens of a sequence, ``step`` for one or a few of each.  ``mass`` is the attention weight that every cached token collects
from a prompt's tokens; ``evict`` gives a row the tokens of another one that hold the most of it.

``run`` computes each in elementary torch operations, or calls the framework where ``own`` is true; ``exact`` states them in 64 bits.
"""
import math

import numpy as np
import torch

own = False
F32, F64 = torch.float32, torch.float64


def listed():
    return [
        # three chat turns that arrive together, a 1B model's heads, capped scores: a call whose time is latency
        dict(name="prompt-turns", kind="prompt", heads=32, kv=8, dim=64, count=3, low=37, high=181, held=0, mask="causal", span=0, cap=50.0, alibi=False,
             evicted=False, lse=False),
        # one document to be read, an 8B model's heads, capped scores, lse for the mass that follows: the largest call
        dict(name="prompt-document", kind="prompt", heads=32, kv=8, dim=128, count=1, low=8192, high=8192, held=0, mask="causal", span=0, cap=50.0, alibi=False,
             evicted=False, lse=True),
        # documents packed behind one another into two rows, distance bias
        dict(name="prompt-packed", kind="prompt", heads=32, kv=8, dim=64, count=2, low=2901, high=4096, held=0, mask="documents", span=700, cap=0.0, alibi=True,
             evicted=False, lse=False),
        # the next portion of long conversations whose caches have been thinned out, windowed, wide heads
        dict(name="prompt-portion", kind="prompt", heads=16, kv=2, dim=256, count=2, low=411, high=512, held=6000, mask="window", span=4096, cap=0.0, alibi=True,
             evicted=True, lse=False),
        # a single token of one sequence: latency
        dict(name="step-one", kind="step", heads=32, kv=8, dim=64, count=1, low=701, high=701, tokens=1, mask="causal", span=0, cap=50.0, alibi=False, evicted=False,
             mass=False),
        # a loaded server's step over ragged contexts that keeps the mass up to date
        dict(name="step-batch", kind="step", heads=32, kv=8, dim=128, count=48, low=600, high=9000, tokens=1, mask="causal", span=0, cap=0.0, alibi=True, evicted=True,
             mass=True),
        # few sequences with very long contexts
        dict(name="step-long", kind="step", heads=32, kv=8, dim=128, count=2, low=99001, high=131000, tokens=1, mask="causal", span=0, cap=30.0, alibi=False,
             evicted=False, mass=True),
        # drafted tokens of eight particles verified in one call, windowed
        dict(name="step-verify", kind="step", heads=32, kv=8, dim=128, count=8, low=3901, high=4203, tokens=9, mask="window", span=2048, cap=0.0, alibi=False,
             evicted=False, mass=False),
        # which tokens a prompt has looked at, the prompt whole
        dict(name="mass-prompt", kind="mass", heads=32, kv=8, dim=128, count=1, low=4096, high=4096, held=0, mask="causal", span=0, cap=50.0, alibi=False, evicted=False),
        # the same by the last tokens of long prompts
        dict(name="mass-tail", kind="mass", heads=32, kv=8, dim=64, count=4, low=33, high=64, held=20000, mask="causal", span=0, cap=0.0, alibi=True, evicted=False),
        # running sequences brought back to their budget
        dict(name="evict-step", kind="evict", kv=8, count=16, low=2100, high=2176, forks=1, keep=2048, first=4, last=256),
        # a long prompt, thinned out, for each of eight particles of two requests
        dict(name="evict-prompt", kind="evict", kv=8, count=2, low=60001, high=65536, forks=8, keep=8192, first=16, last=512),
    ]


def draw(rng):
    def spread(a, b):
        return max(a, min(b, int(math.exp(rng.uniform(math.log(max(a, 1)), math.log(b + 1))))))

    kind = rng.choice(["prompt", "prompt", "step", "step", "mass", "evict"])
    if kind == "evict":
        count, high = rng.randint(1, 24), spread(40, 60000)
        if high > 20000:
            count = min(count, 4)
        keep = spread(8, max(9, high - high // 8))
        first = min(rng.choice([0, 1, 4, 16]), keep // 2)
        return dict(kind="evict", kv=rng.choice([1, 2, 4, 8]), count=count, low=max(1, high - rng.randint(0, high // 3)), high=high, forks=rng.choice([1, 1, 2, 4]),
                    keep=keep, first=first, last=rng.randint(0, keep - first))
    heads, kv, dim = rng.choice([(32, 8, 64), (14, 2, 64), (32, 8, 128), (16, 4, 128), (8, 8, 128), (16, 2, 256)])
    case = dict(kind=kind, heads=heads, kv=kv, dim=dim)
    if kind == "step":
        high, tokens = spread(1, 60000), rng.choice([1, 1, 1, 2, 5, 8])
        count = rng.randint(1, max(1, min(48, 200000 // high)))
        case.update(count=count, low=max(1, high - rng.randint(0, high - 1)), high=high, tokens=tokens)
    else:
        count, high = rng.randint(1, 5), spread(1, 4000)
        held = rng.choice([0, 0, 0, spread(1, 6000)])
        while count * high * (high + held) * heads > 1 << 30:
            high = max(1, high // 2)
        case.update(count=count, low=rng.randint(max(1, high // 3), high), high=high, held=held)
    mask = rng.choice(["causal", "causal", "window", "documents", "prefix"])
    case.update(mask=mask, span=0 if mask == "causal" else spread(16, 3000), cap=rng.choice([0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.5,
                evicted=rng.random() < 0.3)
    if kind == "step":
        case["mass"] = rng.random() < 0.5
    if kind == "prompt":
        case["lse"] = rng.random() < 0.5
    return case


def _spaced(low, high, count):
    """``count`` sizes from low to high, not in order."""
    r = np.linspace(high, low, count).astype(np.int64)
    return r[np.random.RandomState(count).permutation(count)]


def _layout(case):
    """Where the tokens of an attention case are: (tokens held, new tokens) per sequence, positions of the cached tokens, and first and last
    visible position of each new one."""
    if case["kind"] == "step":
        keys = _spaced(case["low"], case["high"], case["count"])
        new = np.full(case["count"], case["tokens"])
        held = keys - new                                            # below zero: a sequence shorter than its tokens, the first of them are padding
    else:
        new = _spaced(case["low"], case["high"], case["count"])
        held = np.full(case["count"], case["held"])
        keys = held + new
    r, positions, bounds = np.random.RandomState(7), [], []
    for h, n, k in zip(held, new, keys):
        pos = np.cumsum(np.where(np.arange(k) < max(h, 0), r.choice([1, 1, 2, 9], k), 1)) - 1 if case["evicted"] else np.arange(k)
        own_pos = np.concatenate([np.full(n - min(n, k), -1), pos[k - min(n, k):]])
        first, last = np.zeros(n, np.int64), own_pos.copy()
        if case["mask"] == "window":
            first = np.maximum(own_pos - case["span"] + 1, 0)
        elif case["mask"] == "documents":                            # of unequal length, span on average
            ends = np.cumsum(np.concatenate([[0], r.randint(1, 2 * case["span"], 2 + int(pos[-1]) // max(1, case["span"] // 2))]))
            first = ends[np.searchsorted(ends, np.maximum(own_pos, 0), side="right") - 1]
        elif case["mask"] == "prefix":
            last = np.where(own_pos < 0, -1, np.maximum(own_pos, case["span"] - 1))
        positions.append(pos)
        bounds.append(np.stack([first, last], 1))
    return held, new, keys, positions, bounds


def _pages(keys, scattered, g):
    """A block table: consecutive pages for each row, or pages in any order; row 0 is nobody's."""
    total = int(sum(keys))
    order = (torch.randperm(total, generator=g, device="cuda") if scattered else torch.arange(total, device="cuda")).int() + 1
    table = torch.zeros(len(keys) + 1, int(max(keys)) + 16, dtype=torch.int32, device="cuda")
    for i, part in enumerate(order.split([int(k) for k in keys])):
        table[i + 1, :len(part)] = part
    return table, total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "evict":
        return _prepare_evict(case, g)
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    held, new, keys, positions, bounds = _layout(case)
    S, T = len(new), int(new.sum())
    table, total = _pages(keys, case["evicted"] or case["kind"] == "step", g)
    at = np.concatenate([[0], np.cumsum(new)[:-1]])
    s = dict(case=case, S=S, T=T, n_max=int(new.max()), k_max=int(keys.max()), keys=total, heads=heads, kv=kv, dim=dim, table=table)
    s["runs"] = torch.tensor(np.stack([np.arange(S) + 1, held, at, new], 1), dtype=torch.int32, device="cuda")
    s["rows"] = s["runs"][:, 0].contiguous()
    s["lens"] = torch.tensor(keys, dtype=torch.int32, device="cuda")
    s["bounds"] = None if case["mask"] == "causal" else torch.tensor(np.concatenate(bounds), dtype=torch.int32, device="cuda")
    s["key_pos"] = None
    if case["evicted"]:
        s["key_pos"] = torch.zeros_like(table)
        for i, p in enumerate(positions):
            s["key_pos"][i + 1, :len(p)] = torch.tensor(p, dtype=torch.int32)
    # queries and keys after their norms and rotations; some keys attract many queries, as the first tokens and punctuation do; values with an offset per channel
    s["q"] = (1.6 * torch.randn(T, heads * dim, generator=g, device="cuda")).bfloat16()
    k = torch.randn(total + 1, kv * dim, generator=g, device="cuda")
    k *= 1 + 0.8 * (torch.rand(total + 1, 1, generator=g, device="cuda") < 0.05)
    s["k"], s["v"] = k.bfloat16(), (torch.randn(total + 1, kv * dim, generator=g, device="cuda") + 0.5 * torch.randn(kv * dim, generator=g, device="cuda")).bfloat16()
    s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device="cuda") if case["alibi"] else None
    s["scale"] = dim ** -0.5
    s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    s["out"] = torch.zeros(T, heads * dim, dtype=torch.bfloat16, device="cuda")
    s["lse"] = torch.zeros(T, heads, device="cuda") if case["kind"] == "mass" or case.get("lse") else None
    s["mass"] = None
    if case["kind"] == "mass" or case.get("mass"):
        s["mass"] = torch.zeros(S + 1, kv, table.shape[1], device="cuda")
        if case["kind"] == "step":                                   # what earlier steps have left
            s["mass"] += 2 * torch.rand(s["mass"].shape, generator=g, device="cuda") ** 4
    if case["kind"] == "mass":
        s["lse"].copy_(_attend(s, F32, lambda x, m: torch.logsumexp(x.masked_fill(~m, -math.inf), -1))[0])
    return s


def _prepare_evict(case, g):
    n = _spaced(case["low"], case["high"], case["count"])
    S, forks, kv = len(n), case["forks"], case["kv"]
    table, total = _pages(n, True, g)
    width = table.shape[1]
    rows = 1 + S + S * forks
    s = dict(case=case, S=S, n_max=int(n.max()), kv=kv, keep=case["keep"])
    s["table"] = torch.cat([table, torch.zeros(S * forks, width, dtype=torch.int32, device="cuda")])
    s["key_pos"] = torch.zeros_like(s["table"])
    s["key_pos"][:S + 1] = torch.cumsum(1 + (torch.rand(S + 1, width, generator=g, device="cuda") < 0.1).int(), 1) - 1
    # the weight that a cached token collects is spread over orders of magnitude, a few hold most of it
    s["mass"] = torch.zeros(rows, kv, width, device="cuda")
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    lens[1:S + 1] = torch.tensor(n, dtype=torch.int32)
    s["mass"][:S + 1] = torch.exp(2.5 * torch.randn(S + 1, kv, width, generator=g, device="cuda")) * (torch.arange(width, device="cuda") < lens[:S + 1, None, None])
    s["lens"] = lens
    s["src"] = torch.arange(1, S + 1, dtype=torch.int32, device="cuda").repeat_interleave(forks)
    s["dst"] = torch.arange(S + 1, rows, dtype=torch.int32, device="cuda")
    s["refcount"] = torch.ones(total + 1, dtype=torch.int32, device="cuda")
    s["free_stack"], s["free_count"] = torch.zeros(total, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    s["kept"] = torch.zeros(S * forks, case["keep"], dtype=torch.int32, device="cuda")
    s["pages"] = total
    s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    return s


def _attend(s, ft, read):
    """Scores of all new tokens, in a batch padded to the longest, and what ``read(scores, mask)`` makes of them, token by token; with the page ids,
    the lengths and the scores' way back to the tokens."""
    case, S, n, k, kv, dim = s["case"], s["S"], s["n_max"], s["k_max"], s["kv"], s["dim"]
    G, dev = s["heads"] // kv, s["q"].device
    row, held, at, new = s["runs"].long().unbind(1)
    i, j = torch.arange(n, device=dev), torch.arange(k, device=dev)
    keys = held + new
    tok = (at[:, None] + i).clamp(max=s["T"] - 1)
    q = s["q"].view(-1, kv, G, dim)[tok].to(ft).permute(0, 2, 3, 1, 4).reshape(S, kv, G * n, dim)
    pages = torch.where(j < keys[:, None], s["table"][row, :k].long(), 0)
    kk = s["k"].view(-1, kv, dim)[pages].to(ft).permute(0, 2, 3, 1)
    x = ((q @ kk) * s["scale"]).view(S, kv, G, n, k)
    if case["cap"] > 0:
        x = case["cap"] * torch.tanh(x / case["cap"])
    idx = held[:, None] + i
    key_pos = j.expand(S, k) if s["key_pos"] is None else s["key_pos"][row, :k].long()
    pos = torch.where(idx < 0, -1, key_pos.gather(1, idx.clamp(0, k - 1)))
    if s["slopes"] is not None:
        x = x - s["slopes"].to(ft).view(1, kv, G, 1, 1) * (pos[:, :, None] - key_pos[:, None, :]).abs().to(ft).view(S, 1, 1, n, k)
    if s["bounds"] is None:
        first, last = torch.zeros_like(pos), pos
    else:
        first, last = s["bounds"].long()[tok].unbind(-1)
    seen = (key_pos[:, None, :] >= first[..., None]) & (key_pos[:, None, :] <= last[..., None]) & (j < keys[:, None, None]) & (i < new[:, None])[..., None]
    seen = seen.view(S, 1, 1, n, k)
    of = torch.bucketize(torch.arange(s["T"], device=dev), at + new, right=True)
    r = read(x, seen)                                                # [S, kv, G, n, ...]
    back = r.movedim(3, 1)[of, torch.arange(s["T"], device=dev) - at[of]]
    return back.reshape(s["T"], s["heads"], *r.shape[4:]).contiguous(), pages, row


def _plain(s):
    if s["case"]["kind"] == "evict":
        return _plain_evict(s)
    case, S, n, k, kv, dim = s["case"], s["S"], s["n_max"], s["k_max"], s["kv"], s["dim"]
    if case["kind"] == "mass":
        def read(x, seen):
            lse = _padded_lse(s)
            w = torch.where(seen & (lse[..., None] > -math.inf), torch.exp(x - lse[..., None]), 0.0)
            s["mass"][s["runs"][:, 0].long(), :, :k] += w.sum((2, 3))
            return w[..., :1]
        _attend(s, F32, read)
        return s["mass"]

    def read(x, seen):
        x = torch.where(seen, x, -math.inf)
        top = x.amax(-1, keepdim=True)
        top = torch.where(top > -math.inf, top, 0.0)
        e = torch.exp(x - top)
        total = e.sum(-1, keepdim=True)
        w = torch.where(total > 0, e / total, 0.0)
        if s["mass"] is not None:
            s["mass"][s["runs"][:, 0].long(), :, :k] += w.sum((2, 3))
        row, held, at, new = s["runs"].long().unbind(1)
        pages = torch.where(torch.arange(k, device=x.device) < (held + new)[:, None], s["table"][row, :k].long(), 0)
        v = s["v"].view(-1, kv, dim)[pages].float().permute(0, 2, 1, 3)
        o = (w.reshape(S, kv, -1, k) @ v).view(S, kv, -1, n, dim)
        return torch.cat([o, (top + torch.log(total))], -1)

    r, _, _ = _attend(s, F32, read)
    s["out"].copy_(r[..., :dim].reshape(s["T"], -1))
    if s["lse"] is not None:
        s["lse"].copy_(r[..., dim])
    return _outputs(s)


def _padded_lse(s):
    at = s["runs"][:, 2].long()
    tok = (at[:, None] + torch.arange(s["n_max"], device=at.device)).clamp(max=s["T"] - 1)
    return s["lse"][tok].view(s["S"], s["n_max"], s["kv"], -1).permute(0, 2, 3, 1)


def _outputs(s):
    return [t for t in (s["out"], s["lse"], s["mass"]) if t is not None]


def _plain_evict(s):
    case, keep, N = s["case"], s["keep"], s["n_max"]
    src, dst = s["src"].long(), s["dst"].long()
    n, before = s["lens"][src].long()[:, None], s["lens"][dst].long()[:, None]
    j = torch.arange(N, device=src.device)
    score = s["mass"][src, 0, :N]
    for h in range(1, s["kv"]):                                      # the heads' weights are added in their order
        score = score + s["mass"][src, h, :N]
    score = torch.where((j < case["first"]) | (j >= n - case["last"]), math.inf, score)
    score = torch.where(j < n, score, -math.inf)
    best = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :keep]
    if best.shape[1] < keep:
        best = torch.nn.functional.pad(best, (0, keep - best.shape[1]), value=N)
    best = torch.where(torch.arange(keep, device=src.device) < n.clamp(max=keep), best, N).sort(1).values
    there = best < N
    at = torch.where(there, best, 0)
    s["kept"].copy_(torch.where(there, best, -1))
    d = dst[:, None].expand_as(best)
    slot = torch.arange(keep, device=src.device).expand_as(best)
    wide = s["table"].shape[1]
    m = min(keep, wide)
    pages = torch.where(there, s["table"][src[:, None], at], 0)
    for t in (s["table"], s["key_pos"]):
        t[dst, :m] = torch.where(there, t[src[:, None], at], t[d, slot.clamp(max=wide - 1)])[:, :m]
    s["refcount"].index_add_(0, pages.reshape(-1).long(), there.reshape(-1).int())
    moved = torch.where(there[:, None, :], s["mass"][src].gather(2, at[:, None, :].expand(-1, s["kv"], -1)), 0.0)[..., :m]
    rest = torch.arange(wide, device=src.device) < before
    s["mass"][dst] = torch.where(rest[:, None, :], 0.0, s["mass"][dst])
    s["mass"][dst, :, :m] = torch.where(there[:, None, :m], moved, s["mass"][dst, :, :m])
    s["lens"][dst] = n[:, 0].clamp(max=keep).int()
    return [s["kept"], s["table"], s["key_pos"], s["mass"], s["lens"], s["refcount"]]


def run(s):
    if not own:
        return _plain(s)
    from smcsd_b200.ops import native_shaped as N
    kind = s["case"]["kind"]
    if kind == "evict":
        c = s["case"]
        if "work" not in s:                                          # a server keeps one beside its allocator
            s["work"] = torch.zeros(N.evict_work_bytes(s["pages"]), dtype=torch.uint8, device="cuda")
        N.evict_tokens(s["table"], s["src"], s["dst"], s["lens"], s["mass"], s["refcount"], s["free_stack"], s["free_count"], keep=c["keep"], first=c["first"],
                       last=c["last"], key_pos=s["key_pos"], kept=s["kept"], work=s["work"], status=s["status"])
        return [s["kept"], s["table"], s["key_pos"], s["mass"], s["lens"], s["refcount"]]
    shape = dict(Hq=s["heads"], Hkv=s["kv"], D=s["dim"], scale=s["scale"], softcap=s["case"]["cap"], slopes=s["slopes"], bounds=s["bounds"],
                 key_pos=s["key_pos"], status=s["status"])
    if kind == "prompt":
        N.attention_shaped_prompt(s["q"], s["k"], s["v"], s["table"], s["runs"], s["out"], T=s["T"], lse=s["lse"], **shape)
        return _outputs(s)
    if kind == "mass":
        N.attention_key_mass(s["q"], s["k"], s["table"], s["runs"], s["lse"], s["mass"], T=s["T"], **shape)
        return s["mass"]
    E = s["case"]["tokens"]
    if "work" not in s:                                              # a server keeps one for all its steps
        s["work"] = torch.zeros(N.shaped_step_work_bytes(s["S"], E, s["heads"], s["kv"], s["dim"], s["keys"] if s["mass"] is not None else 0),
                                dtype=torch.uint8, device="cuda")
    N.attention_shaped_step(s["q"], s["k"], s["v"], s["table"], s["rows"], s["lens"], s["out"], bs=s["S"], E=E, work=s["work"], lse=s["lse"], mass=s["mass"], **shape)
    return _outputs(s)


def work(case):
    if case["kind"] == "evict":
        n, kept = _spaced(case["low"], case["high"], case["count"]), 0
        kept = int(np.minimum(n, case["keep"]).sum()) * case["forks"]
        # every head's mass of every token once; pages, positions, mass of the kept ones read and written, their counts and indices
        return {"bytes": 4 * case["kv"] * int(n.sum()) + kept * (2 * 8 + 4 * case["kv"] + 12), "flops": case["kv"] * int(n.sum())}
    held, new, keys, positions, bounds = _layout(case)
    pairs, seen = 0, 0
    for p, b in zip(positions, bounds):
        lo, hi = np.searchsorted(p, b[:, 0], side="left"), np.searchsorted(p, b[:, 1], side="right")
        some = hi > lo
        pairs += int((hi - lo)[some].sum())
        if some.any():
            diff = np.zeros(len(p) + 1, np.int64)
            np.add.at(diff, lo[some], 1)
            np.add.at(diff, hi[some], -1)
            seen += int((np.cumsum(diff)[:-1] > 0).sum())
    T, row, kv_row = int(new.sum()), 2 * case["heads"] * case["dim"], 2 * case["kv"] * case["dim"]
    if case["kind"] == "mass":
        return {"bytes": T * row + 4 * T * case["heads"] + seen * (kv_row + 4 + 8 * case["kv"]), "flops": 2 * case["dim"] * case["heads"] * pairs}
    extra = (4 * T * case["heads"] if case.get("lse") else 0) + (8 * case["kv"] * seen if case.get("mass") else 0) + (4 * seen if case["evicted"] else 0)
    return {"bytes": 2 * T * row + seen * (2 * kv_row + 4) + extra, "flops": 4 * case["dim"] * case["heads"] * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "evict":
        return _exact_evict(s)
    kv, dim = s["kv"], s["dim"]
    G = s["heads"] // kv
    out, lse = torch.zeros(s["T"], s["heads"], dim, dtype=F64, device="cuda"), torch.full((s["T"], s["heads"]), -math.inf, dtype=F64, device="cuda")
    mass = None if s["mass"] is None else s["mass"].double()
    for row, held, at, n in s["runs"].tolist():
        L = held + n
        pages = s["table"][row, :L].long()
        pos = torch.arange(L, device="cuda") if s["key_pos"] is None else s["key_pos"][row, :L].long()
        lead = max(0, -held)                                         # padding ahead of a short sequence sees nothing
        mine = pos[max(held, 0):]
        lo, hi = (torch.zeros_like(mine), mine) if s["bounds"] is None else s["bounds"][at + lead:at + n].long().unbind(1)
        hidden = (pos < lo[:, None]) | (pos > hi[:, None])
        empty = hidden.all(1)
        for h in range(s["heads"]):
            c = slice(h // G * dim, (h // G + 1) * dim)
            z = s["q"][at + lead:at + n, h * dim:(h + 1) * dim].double() @ s["k"][pages, c].double().T * s["scale"]
            if case["cap"] > 0:
                z = torch.tanh(z / case["cap"]) * case["cap"]
            if s["slopes"] is not None:
                z = z - s["slopes"][h].double() * (mine[:, None] - pos).abs()
            z = z.masked_fill(hidden, -math.inf)
            if case["kind"] == "mass":
                total = s["lse"][at + lead:at + n, h].double()[:, None]
            else:
                total = torch.logsumexp(z, 1, keepdim=True)
            w = torch.exp(z - total).masked_fill(empty[:, None], 0.0)
            if mass is not None:
                mass[row, h // G, :L] += w.sum(0)
            if case["kind"] != "mass":
                out[at + lead:at + n, h] = w @ s["v"][pages, c].double()
                lse[at + lead:at + n, h] = total[:, 0]
    if case["kind"] == "mass":
        return mass
    return [t for t in (out.view(s["T"], -1), lse if s["lse"] is not None else None, mass) if t is not None]


def _exact_evict(s):
    case = s["case"]
    mass, table, pos = s["mass"].double().cpu().numpy(), s["table"].cpu().numpy(), s["key_pos"].cpu().numpy()
    lens, refs, kept = s["lens"].cpu().numpy(), s["refcount"].cpu().numpy(), s["kept"].cpu().numpy()
    for f, (a, b) in enumerate(zip(s["src"].tolist(), s["dst"].tolist())):
        n = int(lens[a])
        take = np.arange(n)
        if n > case["keep"]:
            score = np.zeros(n, np.float32)                          # the operator's score is the 32-bit sum over the heads in their order
            for h in range(s["kv"]):
                score = (score.astype(np.float64) + mass[a, h, :n]).astype(np.float32)
            inner = np.arange(case["first"], n - case["last"])
            chosen = inner[np.lexsort((inner, -score[inner]))[:case["keep"] - case["first"] - case["last"]]]
            take = np.sort(np.concatenate([np.arange(case["first"]), chosen, np.arange(n - case["last"], n)]))
        m = len(take)
        kept[f] = -1
        kept[f, :m] = take
        mass[b, :, :lens[b]] = 0
        table[b, :m], pos[b, :m], mass[b, :, :m], lens[b] = table[a, take], pos[a, take], mass[a][:, take], m
        np.add.at(refs, table[a, take], 1)
    return [kept, table, pos, mass, lens, refs]
