"""Attention over the paged cache whose scores are capped, lowered by distance or masked to intervals, and a cache held to a budget.

With x = scale q.k, then ``softcap`` tanh(x / softcap) where ``softcap`` > 0, then x - slopes[head] |distance| where ``slopes`` are given,
a token attends the cached tokens whose positions lie in its interval ``bounds[t]`` = (first, last), both included; without
``bounds`` all up to its own.  ``score_bounds`` makes the intervals of windows, packed documents and prefixes.  A token that sees nothing gets zeros
and a log-sum-exp of -inf.

    attention_shaped_prompt    many tokens of a sequence
    attention_shaped_step      the last one or few of each
    attention_key_mass         the weight that every cached token collects from a prompt's tokens
    evict_tokens               the tokens that collected most stay, the others give their pages back

The cache is the block table's: one page per token, bf16 rows of Hkv * D values (the e4m3 cache is refused), all tokens of a call
already written.  ``key_pos`` lists the positions of a row's tokens, ascending and below 2^24, once tokens have been shed; without it token j
of a row has position j.  The weights live in ``mass`` [rows, Hkv, tokens], fp32, beside the block table; entries behind a row's last
token are zero.  A key or value that is not finite spoils the tokens that share a tile of queries with one that sees it; tokens
that nobody sees are not read.

As everywhere, calls run on the current stream, allocate nothing and can be captured; ``status`` collects error bits.  Two calls that may
run at the same time need a workspace each.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import native as K

_BF16, _I32, _F32, _U8 = torch.bfloat16, torch.int32, torch.float32, torch.uint8
_lib = None


def _library():
    global _lib
    if _lib is None:
        L, vp, i, ll, f = K.lib(), C.c_void_p, C.c_int, C.c_longlong, C.c_float
        L.smc_shaped_prompt.argtypes = [vp, ll, vp, vp, i, vp, i, i, vp, i, vp, i, vp, ll, vp, i, i, i, i, f, f, vp, vp, vp, i, vp]
        L.smc_shaped_step.argtypes = [vp, ll, vp, vp, i, vp, i, i, vp, i, vp, vp, vp, ll, vp, vp, ll, i, i, i, i, i, f, f, vp, vp, vp, ll, vp, i, vp]
        L.smc_shaped_mass.argtypes = [vp, ll, vp, i, vp, i, i, vp, i, vp, i, vp, vp, ll, i, i, i, i, f, f, vp, vp, vp, i, vp]
        L.smc_evict.argtypes = [vp, ll, vp, ll, vp, ll, vp, i, vp, vp, i, i, i, i, i, vp, vp, vp, vp, i, vp, ll, vp, vp]
        L.smc_shaped_step_work.argtypes = [i, i, i, i, i, ll]
        L.smc_evict_work.argtypes = [i]
        for name in ("smc_shaped_prompt", "smc_shaped_step", "smc_shaped_mass", "smc_evict"):
            getattr(L, name).restype = i
        L.smc_shaped_step_work.restype = L.smc_evict_work.restype = ll
        _lib = L
    return _lib


def _is(t: torch.Tensor, name: str, dtype: torch.dtype, device, shape=None) -> int:
    """Address of a tensor of this type on this device whose last axis is contiguous; ``shape``: at least these sizes, all axes contiguous."""
    if t.dtype is not dtype or t.device != device:
        raise ValueError(f"{name}: {dtype} on {device} expected, got {t.dtype} on {t.device}")
    if shape is not None:
        if t.dim() != len(shape) or not t.is_contiguous() or any(a < b for a, b in zip(t.shape, shape)) or t.shape[1:] != shape[1:]:
            raise ValueError(f"{name}: contiguous {tuple(shape)} expected, got {tuple(t.shape)} with strides {t.stride()}")
    elif t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}: the last axis has to be contiguous, got strides {t.stride()}")
    return t.data_ptr()


def _table(t: Optional[torch.Tensor], name: str, device, rows: int, cols: int):
    """Address and row stride of an int32 table of at least ``rows`` x ``cols``, or nothing."""
    if t is None:
        return None, 0
    p = _is(t, name, _I32, device)
    if t.dim() != 2 or t.shape[0] < rows or t.shape[1] < cols:
        raise ValueError(f"{name}: at least [{rows}, {cols}] expected, got {tuple(t.shape)}")
    return p, t.stride(0)


def _device(q: torch.Tensor):
    device = q.device
    if device.type != "cuda" or device.index != torch._C._cuda_getDevice():
        raise ValueError(f"tensors on the current CUDA device expected, got {device}")
    return device


def _rows(t: torch.Tensor, name: str, device, T: int, width: int):
    """Address and stride of T rows of ``width`` bf16 values."""
    p = _is(t, name, _BF16, device)
    if t.dim() != 2 or t.shape[0] < T or t.shape[1] != width:
        raise ValueError(f"{name}: at least [{T}, {width}] expected, got {tuple(t.shape)}")
    return p, t.stride(0)


def _pool(t: torch.Tensor, name: str, device, width: int) -> int:
    if t.dim() != 2 or t.shape[1] != width:
        raise ValueError(f"{name}: [pages + 1, {width}] expected, got {tuple(t.shape)}")
    return _is(t, name, _BF16, device, t.shape)


def _weights(mass: torch.Tensor, device, rows: int, Hkv: int, cols: int):
    p = _is(mass, "mass", _F32, device)
    if mass.dim() != 3 or mass.shape[0] < rows or mass.shape[1] != Hkv or mass.shape[2] < cols or mass.stride(0) != Hkv * mass.stride(1):
        raise ValueError(f"mass: at least [{rows}, {Hkv}, {cols}], heads of a row behind one another, expected, got {tuple(mass.shape)} with strides {mass.stride()}")
    return p, mass.stride(1)


def _shape(device, T, Hq, slopes, bounds, status):
    return (None if slopes is None else _is(slopes, "slopes", _F32, device, (Hq,)), None if bounds is None else _is(bounds, "bounds", _I32, device, (T, 2)),
            _is(status, "status", _I32, device))


def score_bounds(positions: torch.Tensor, *, window: int = 0, doc_first: Optional[torch.Tensor] = None, prefix: Optional[torch.Tensor] = None) -> torch.Tensor:
    """First and last visible position [T, 2] int32 of tokens at ``positions`` [T]: all up to their own, of them the last ``window`` (0: all) from the
    first token of their document (``doc_first`` [T], positions) on; tokens in front of ``prefix`` ([T] or a number: positions
    below it) also see the rest of the prefix.  A window or a document that cuts the prefix cuts it for the tokens inside too."""
    pos = positions.to(torch.int64)
    first = torch.zeros_like(pos) if window <= 0 else (pos - window + 1).clamp(min=0)
    if doc_first is not None:
        first = torch.maximum(first, doc_first.to(first))
    last = pos if prefix is None else torch.maximum(pos, torch.as_tensor(prefix, device=pos.device).to(pos) - 1)
    return torch.stack([first, last], 1).to(_I32)


def attention_shaped_prompt(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor, runs: torch.Tensor, out: torch.Tensor, *,
                            T: int, Hq: int, Hkv: int, D: int, scale: float, status: torch.Tensor, softcap: float = 0.0,
                            slopes: Optional[torch.Tensor] = None, bounds: Optional[torch.Tensor] = None, key_pos: Optional[torch.Tensor] = None,
                            lse: Optional[torch.Tensor] = None, pdl: bool = False) -> None:
    """Rotated queries ``q`` [T, Hq * D] of whole prompts or portions of them -> ``out`` [T, Hq * D] and ``lse`` [T, Hq].  ``runs`` [n, 4] int32 on the
    device: block-table row, tokens held before, index of the first new token in ``q``, new tokens; rows of ``out`` that no run
    names are left alone.  Heads of 64, 128 or 256, at most 128 query heads to a KV head."""
    L, dev = _library(), _device(q)
    (qp, ldq), (op, ldo) = _rows(q, "q", dev, T, Hq * D), _rows(out, "out", dev, T, Hq * D)
    bt, bts = _table(block_table, "block_table", dev, 1, 1)
    kp, kps = _table(key_pos, "key_pos", dev, block_table.shape[0], block_table.shape[1])
    sl, bo, st = _shape(dev, T, Hq, slopes, bounds, status)
    K._check(L.smc_shaped_prompt(qp, ldq, _pool(k_pool, "k_pool", dev, Hkv * D), _pool(v_pool, "v_pool", dev, Hkv * D), min(k_pool.shape[0], v_pool.shape[0]) - 1,
                                 bt, block_table.shape[1] if block_table.shape[0] == 1 else bts, block_table.shape[0], kp, kps,
                                 _is(runs, "runs", _I32, dev, (runs.shape[0], 4)), runs.shape[0], op, ldo,
                                 None if lse is None else _is(lse, "lse", _F32, dev, (T, Hq)), T, Hq, Hkv, D, scale, softcap, sl, bo, st, int(pdl), K._stream()),
             "smc_shaped_prompt")


def attention_key_mass(q: torch.Tensor, k_pool: torch.Tensor, block_table: torch.Tensor, runs: torch.Tensor, lse: torch.Tensor, mass: torch.Tensor, *, T: int,
                       Hq: int, Hkv: int, D: int, scale: float, status: torch.Tensor, softcap: float = 0.0, slopes: Optional[torch.Tensor] = None,
                       bounds: Optional[torch.Tensor] = None, key_pos: Optional[torch.Tensor] = None, pdl: bool = False) -> None:
    """``mass[row, kv head, j]`` += the attention weight that token j of the row gets from the tokens and query heads of the pass that left ``lse``
    (same arguments).  ``runs`` may list fewer tokens than that pass - the last ones of a prompt, say - but a row only once."""
    L, dev = _library(), _device(q)
    qp, ldq = _rows(q, "q", dev, T, Hq * D)
    bt, bts = _table(block_table, "block_table", dev, 1, 1)
    kp, kps = _table(key_pos, "key_pos", dev, block_table.shape[0], block_table.shape[1])
    sl, bo, st = _shape(dev, T, Hq, slopes, bounds, status)
    mp, ms = _weights(mass, dev, block_table.shape[0], Hkv, block_table.shape[1])
    K._check(L.smc_shaped_mass(qp, ldq, _pool(k_pool, "k_pool", dev, Hkv * D), k_pool.shape[0] - 1, bt, block_table.shape[1] if block_table.shape[0] == 1 else bts,
                               block_table.shape[0], kp, kps, _is(runs, "runs", _I32, dev, (runs.shape[0], 4)), runs.shape[0], _is(lse, "lse", _F32, dev, (T, Hq)),
                               mp, ms, T, Hq, Hkv, D, scale, softcap, sl, bo, st, int(pdl), K._stream()), "smc_shaped_mass")


def shaped_step_work_bytes(bs: int, E: int, Hq: int, Hkv: int, D: int, keys: int = 0) -> int:
    """Bytes of workspace for ``attention_shaped_step`` (uint8, zeros at first; a larger one serves smaller batches).  With the mass: ``keys``,
    the cached tokens of all sequences of a step together."""
    n = _library().smc_shaped_step_work(bs, E, Hq, Hkv, D, keys)
    if n < 0:
        raise ValueError(f"no step for {bs} sequences of {E} tokens with {Hq} heads of {D} on {Hkv} KV heads")
    return n


def attention_shaped_step(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor, rows: torch.Tensor, lens: torch.Tensor,
                          out: torch.Tensor, *, bs: int, E: int, Hq: int, Hkv: int, D: int, scale: float, status: torch.Tensor, work: torch.Tensor,
                          softcap: float = 0.0, slopes: Optional[torch.Tensor] = None, bounds: Optional[torch.Tensor] = None,
                          key_pos: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None, mass: Optional[torch.Tensor] = None, pdl: bool = False) -> None:
    """The last E of the ``lens[s]`` cached tokens of each sequence (``rows``, ``lens`` [bs] int32; a sequence shorter than E is padded in front): queries ``q``
    [bs * E, Hq * D] -> ``out`` and ``lse``.  With ``mass`` (rows listed once) the weights of the step are added to it.  At most 64 rows E * Hq / Hkv, 1024 sequences;
    ``work``: see ``shaped_step_work_bytes``."""
    L, dev, T = _library(), _device(q), bs * E
    (qp, ldq), (op, ldo) = _rows(q, "q", dev, T, Hq * D), _rows(out, "out", dev, T, Hq * D)
    bt, bts = _table(block_table, "block_table", dev, 1, 1)
    kp, kps = _table(key_pos, "key_pos", dev, block_table.shape[0], block_table.shape[1])
    sl, bo, st = _shape(dev, T, Hq, slopes, bounds, status)
    mp, ms = (None, 0) if mass is None else _weights(mass, dev, block_table.shape[0], Hkv, block_table.shape[1])
    K._check(L.smc_shaped_step(qp, ldq, _pool(k_pool, "k_pool", dev, Hkv * D), _pool(v_pool, "v_pool", dev, Hkv * D), min(k_pool.shape[0], v_pool.shape[0]) - 1, bt,
                               block_table.shape[1] if block_table.shape[0] == 1 else bts, block_table.shape[0], kp, kps, _is(rows, "rows", _I32, dev, (bs,)),
                               _is(lens, "lens", _I32, dev, (bs,)), op, ldo, None if lse is None else _is(lse, "lse", _F32, dev, (T, Hq)), mp, ms, bs, E, Hq, Hkv, D,
                               scale, softcap, sl, bo, _is(work, "work", _U8, dev, work.shape), work.numel(), st, int(pdl), K._stream()),
             "smc_shaped_step")


def evict_work_bytes(n_pages: int) -> int:
    """Bytes of workspace for ``evict_tokens`` on an allocator of ``n_pages`` pages (uint8, zeros at first)."""
    return _library().smc_evict_work(n_pages)


def evict_tokens(block_table: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, lens: torch.Tensor, mass: torch.Tensor, refcount: torch.Tensor,
                 free_stack: torch.Tensor, free_count: torch.Tensor, *, keep: int, first: int, last: int, kept: torch.Tensor, work: torch.Tensor,
                 status: torch.Tensor, key_pos: Optional[torch.Tensor] = None) -> None:
    """Of the ``lens[row]`` tokens of each row in ``src`` [n] the first ``first``, the last ``last`` and those between with the highest sum of ``mass`` over the KV
    heads stay, at most ``keep`` in all (equal sums: the lower index).  They move, in their order, with page, position and weights to the row
    in ``dst``: the same one, whose other tokens give up their pages' references, or another, free one, which takes references.  ``lens`` [rows]
    is updated, ``kept`` [n, keep] receives the indices (-1 behind the last).  Weights behind the kept tokens are cleared up to the old length of the row; its other
    entries there are left as they were.  A row may be written by one entry only, and then be read by no other."""
    L, dev = _library(), _device(block_table)
    R, n = block_table.shape[0], src.shape[0]
    bt, bts = _table(block_table, "block_table", dev, 1, 1)
    cols = block_table.shape[1]
    if bts < cols and R > 1:
        raise ValueError(f"block_table: rows may not overlap, got strides {block_table.stride()}")
    kp, kps = _table(key_pos, "key_pos", dev, R, cols)
    mp, ms = _weights(mass, dev, R, mass.shape[1], cols)
    pages = refcount.shape[0] - 1
    if free_stack.shape[0] < pages:
        raise ValueError(f"free_stack: room for {pages} pages expected, got {free_stack.shape[0]}")
    K._check(L.smc_evict(bt, bts if R > 1 else cols, kp, kps if R > 1 else max(kps, cols), mp, ms, _is(lens, "lens", _I32, dev, (R,)), R, _is(src, "src", _I32, dev, (n,)),
                         _is(dst, "dst", _I32, dev, (n,)), n, mass.shape[1], keep, first, last, _is(kept, "kept", _I32, dev, (n, keep)),
                         _is(refcount, "refcount", _I32, dev, refcount.shape), _is(free_stack, "free_stack", _I32, dev, free_stack.shape),
                         _is(free_count, "free_count", _I32, dev, free_count.shape), pages, _is(work, "work", _U8, dev, work.shape), work.numel(),
                         _is(status, "status", _I32, dev), K._stream()), "smc_evict")
