"""Attention over the paged cache whose scores are capped, lowered by distance or masked to intervals, and a cache held to a budget.

With x = scale q.k, then ``softcap`` tanh(x / softcap) where ``softcap`` > 0, then x - slopes[head] |distance| where ``slopes`` are given,
a token attends the cached tokens whose positions lie in its interval ``bounds[t]`` = (first, last), both included; without
``bounds`` all up to its own.  ``score_bounds`` makes the intervals of windows, packed documents and prefixes.  A token that sees nothing gets zeros
and a log-sum-exp of -inf.  ``scale``, ``softcap`` and ``scale / softcap`` have to lie within the range of normal fp32 numbers, or the call is refused.

    attention_shaped_prompt    many tokens of a sequence
    attention_shaped_step      the last one or few of each
    attention_key_mass         the weight that every cached token collects from a prompt's tokens
    evict_tokens               the tokens that collected most stay, the others give their pages back

The cache is the block table's: one page per token, bf16 rows of Hkv * D values (the e4m3 cache is refused), all tokens of a call
already written.  ``key_pos`` lists the positions of a row's tokens, ascending and below 2^24, once tokens have been shed; without it token j
of a row has position j.  The weights live in ``mass`` [rows, Hkv, tokens], fp32, beside the block table; entries behind a row's last
token are zero.  A key or value that is not finite spoils the tokens that share a tile of queries with one that sees
it (prompts: up to 256 rows of tokens x heads, 128 with heads of 256; steps: those of the sequence); cached tokens outside the span of a tile's intervals are not read.

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
        L.smc_shaped_prompt.argtypes = [vp, ll, vp, vp, i, vp, ll, i, vp, i, vp, i, vp, ll, vp, i, i, i, i, f, f, vp, vp, vp, i, vp]
        L.smc_shaped_step.argtypes = [vp, ll, vp, vp, i, vp, ll, i, vp, i, vp, vp, vp, ll, vp, vp, ll, i, i, i, i, i, f, f, vp, vp, vp, ll, vp, i, vp]
        L.smc_shaped_mass.argtypes = [vp, ll, vp, i, vp, ll, i, vp, i, vp, i, vp, vp, ll, i, i, i, i, f, f, vp, vp, vp, i, vp]
        L.smc_evict.argtypes = [vp, ll, vp, ll, vp, ll, vp, i, vp, vp, i, i, i, i, i, vp, vp, vp, vp, i, vp, ll, vp, vp]
        L.smc_shaped_step_work.argtypes = [i, i, i, i, i, ll]
        L.smc_evict_work.argtypes = [i]
        for name in ("smc_shaped_prompt", "smc_shaped_step", "smc_shaped_mass", "smc_evict"):
            getattr(L, name).restype = i
        L.smc_shaped_step_work.restype = L.smc_evict_work.restype = ll
        K._KERNELS_PER_CALL.update({"smc_evict": 2, "smc_shaped_step with mass": 2})
        _lib = L
    return _lib


def _wrong(t: torch.Tensor, name: str, want: str):
    return ValueError(f"{name}: {want} expected, got {t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device}")


def _flat(t: torch.Tensor, name: str, dtype: torch.dtype, dev: int, shape) -> int:
    """Address of a contiguous tensor of this type on this device, at least ``shape[0]`` long and of those further sizes."""
    got = t.shape
    if t.dtype is not dtype or t.get_device() != dev or len(got) != len(shape) or got[0] < shape[0] or got[1:] != shape[1:] or not t.is_contiguous():
        raise _wrong(t, name, f"contiguous {dtype} {tuple(shape)} on cuda:{dev}")
    return t.data_ptr()


def _device(q: torch.Tensor) -> int:
    dev = q.get_device()
    if dev < 0 or dev != torch._C._cuda_getDevice():
        raise ValueError(f"tensors on the current CUDA device expected, got {q.device}")
    return dev


def _rows(t: torch.Tensor, name: str, dev: int, T: int, width: int):
    """Address and stride of at least T rows of ``width`` bf16 values."""
    got, stride = t.shape, t.stride()
    if t.dtype is not _BF16 or t.get_device() != dev or len(got) != 2 or got[0] < T or got[1] != width or stride[1] != 1:
        raise _wrong(t, name, f"at least {T} rows of {width} bfloat16 values on cuda:{dev}")
    return t.data_ptr(), stride[0]


def _pool(t: torch.Tensor, name: str, dev: int, width: int) -> int:
    if t.dtype is not _BF16 or t.get_device() != dev or t.dim() != 2 or t.shape[0] < 1 or t.shape[1] != width or not t.is_contiguous():
        raise _wrong(t, name, f"contiguous bfloat16 [pages + 1, {width}] on cuda:{dev}")
    return t.data_ptr()


def _tables(block_table: torch.Tensor, key_pos: Optional[torch.Tensor], dev: int):
    """Address, pitch (row stride, columns above bit 32) and rows of the block table, address and row stride of the positions."""
    shape, stride = block_table.shape, block_table.stride()
    if block_table.dtype is not _I32 or block_table.get_device() != dev or len(shape) != 2 or shape[0] < 1 or shape[1] < 1 or stride[1] != 1 or stride[0] < shape[1] and shape[0] > 1:
        raise _wrong(block_table, "block_table", f"int32 [rows, tokens] on cuda:{dev}")
    rows, cols = shape
    bt = (block_table.data_ptr(), (stride[0] if rows > 1 else cols) | cols << 32, rows)
    if key_pos is None:
        return bt, (None, 0)
    stride = key_pos.stride()
    if key_pos.dtype is not _I32 or key_pos.get_device() != dev or key_pos.dim() != 2 or key_pos.shape[0] < rows or key_pos.shape[1] < cols or stride[1] != 1 or stride[0] < cols:
        raise _wrong(key_pos, "key_pos", f"int32, at least [{rows}, {cols}], on cuda:{dev}")
    return bt, (key_pos.data_ptr(), stride[0])


def _weights(mass: torch.Tensor, dev: int, rows: int, Hkv: int, cols: int):
    shape, stride = mass.shape, mass.stride()
    if mass.dtype is not _F32 or mass.get_device() != dev or len(shape) != 3 or shape[0] < rows or shape[1] != Hkv or shape[2] < cols or stride[2] != 1 \
            or stride[1] < shape[2] or stride[0] != Hkv * stride[1]:
        raise _wrong(mass, "mass", f"float32, at least [{rows}, {Hkv}, {cols}], the heads of a row behind one another, on cuda:{dev}")
    return mass.data_ptr(), stride[1]


def _shape(dev, T, Hq, slopes, bounds, status):
    return (None if slopes is None else _flat(slopes, "slopes", _F32, dev, (Hq,)), None if bounds is None else _flat(bounds, "bounds", _I32, dev, (T, 2)),
            _flat(status, "status", _I32, dev, (1,)))


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
    device: block-table row, tokens held before, index of the first new token in ``q``, new tokens (no token of ``q`` in two runs); rows of ``out`` that no run
    names are left alone.  Heads of 64, 128 or 256, at most 128 query heads to a KV head."""
    L, dev, width = _library(), _device(q), Hkv * D
    (qp, ldq), (op, ldo) = _rows(q, "q", dev, T, Hq * D), _rows(out, "out", dev, T, Hq * D)
    (bt, bts, rows), (kp, kps) = _tables(block_table, key_pos, dev)
    sl, bo, st = _shape(dev, T, Hq, slopes, bounds, status)
    n = runs.shape[0]
    K._check(L.smc_shaped_prompt(qp, ldq, _pool(k_pool, "k_pool", dev, width), _pool(v_pool, "v_pool", dev, width), min(k_pool.shape[0], v_pool.shape[0]) - 1, bt, bts, rows,
                                 kp, kps, _flat(runs, "runs", _I32, dev, (n, 4)), n, op, ldo, None if lse is None else _flat(lse, "lse", _F32, dev, (T, Hq)), T, Hq, Hkv, D,
                                 scale, softcap, sl, bo, st, pdl, K._stream()), "smc_shaped_prompt")


def attention_key_mass(q: torch.Tensor, k_pool: torch.Tensor, block_table: torch.Tensor, runs: torch.Tensor, lse: torch.Tensor, mass: torch.Tensor, *, T: int,
                       Hq: int, Hkv: int, D: int, scale: float, status: torch.Tensor, softcap: float = 0.0, slopes: Optional[torch.Tensor] = None,
                       bounds: Optional[torch.Tensor] = None, key_pos: Optional[torch.Tensor] = None, pdl: bool = False) -> None:
    """``mass[row, kv head, j]`` += the attention weight that token j of the row gets from the tokens and query heads of the pass that left ``lse``
    (same arguments).  ``runs`` may list fewer tokens than that pass - the last ones of a prompt, say - but a row only once, and tokens of the row behind the last listed
    one get nothing."""
    L, dev = _library(), _device(q)
    qp, ldq = _rows(q, "q", dev, T, Hq * D)
    (bt, bts, rows), (kp, kps) = _tables(block_table, key_pos, dev)
    sl, bo, st = _shape(dev, T, Hq, slopes, bounds, status)
    mp, ms = _weights(mass, dev, rows, Hkv, block_table.shape[1])
    n = runs.shape[0]
    K._check(L.smc_shaped_mass(qp, ldq, _pool(k_pool, "k_pool", dev, Hkv * D), k_pool.shape[0] - 1, bt, bts, rows, kp, kps, _flat(runs, "runs", _I32, dev, (n, 4)), n,
                               _flat(lse, "lse", _F32, dev, (T, Hq)), mp, ms, T, Hq, Hkv, D, scale, softcap, sl, bo, st, pdl, K._stream()), "smc_shaped_mass")


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
    L, dev, T, width = _library(), _device(q), bs * E, Hkv * D
    (qp, ldq), (op, ldo) = _rows(q, "q", dev, T, Hq * D), _rows(out, "out", dev, T, Hq * D)
    (bt, bts, n), (kp, kps) = _tables(block_table, key_pos, dev)
    sl, bo, st = _shape(dev, T, Hq, slopes, bounds, status)
    mp, ms = (None, 0) if mass is None else _weights(mass, dev, n, Hkv, block_table.shape[1])
    rc = L.smc_shaped_step(qp, ldq, _pool(k_pool, "k_pool", dev, width), _pool(v_pool, "v_pool", dev, width), min(k_pool.shape[0], v_pool.shape[0]) - 1, bt, bts, n, kp, kps,
                           _flat(rows, "rows", _I32, dev, (bs,)), _flat(lens, "lens", _I32, dev, (bs,)), op, ldo, None if lse is None else _flat(lse, "lse", _F32, dev, (T, Hq)),
                           mp, ms, bs, E, Hq, Hkv, D, scale, softcap, sl, bo, _flat(work, "work", _U8, dev, (1,)), work.numel(), st, pdl, K._stream())
    K._check(rc, "smc_shaped_step" if mass is None else "smc_shaped_step with mass")


def evict_work_bytes(n_pages: int) -> int:
    """Bytes of workspace for ``evict_tokens`` on an allocator of ``n_pages`` pages (uint8, zeros at first)."""
    n = _library().smc_evict_work(n_pages)
    if n < 0:
        raise ValueError(f"no allocator of {n_pages} pages")
    return n


def evict_tokens(block_table: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, lens: torch.Tensor, mass: torch.Tensor, refcount: torch.Tensor,
                 free_stack: torch.Tensor, free_count: torch.Tensor, *, keep: int, first: int, last: int, kept: torch.Tensor, work: torch.Tensor,
                 status: torch.Tensor, key_pos: Optional[torch.Tensor] = None) -> None:
    """Of the ``lens[row]`` tokens of each row in ``src`` [n] the first ``first``, the last ``last`` and those between with the highest sum of ``mass`` over the KV
    heads stay, at most ``keep`` in all (equal sums: the lower index).  They move, in their order, with page, position and weights to the row
    in ``dst``: the same one, whose other tokens give up their pages' references, or another, free one, which takes references.  Without ``key_pos`` they are known by their
    new indices from then on, which is right for attention without ``bounds`` and ``slopes`` only.  ``lens`` [rows]
    is updated, ``kept`` [n, keep] receives the indices (-1 behind the last).  Weights behind the kept tokens are cleared up to the old length of the row; its other
    entries there are left as they were.  A row may be written by one entry only, and then be read by no other.  At most 4096 entries, block tables of at most 262144 columns
    (one of more is handed over as a slice of them)."""
    L, dev = _library(), _device(block_table)
    if src.shape[0] > 4096 or block_table.dim() == 2 and block_table.shape[1] > 262144:
        raise ValueError(f"at most 4096 entries and 262144 columns of a block table expected, got {src.shape[0]} and {block_table.shape[1]}")
    (bt, bts, R), (kp, kps) = _tables(block_table, key_pos, dev)
    n, heads, pages = src.shape[0], mass.shape[1], refcount.shape[0] - 1
    mp, ms = _weights(mass, dev, R, heads, block_table.shape[1])
    K._check(L.smc_evict(bt, bts, kp, kps, mp, ms, _flat(lens, "lens", _I32, dev, (R,)), R, _flat(src, "src", _I32, dev, (n,)), _flat(dst, "dst", _I32, dev, (n,)), n, heads, keep,
                         first, last, _flat(kept, "kept", _I32, dev, (n, keep)), _flat(refcount, "refcount", _I32, dev, (pages + 1,)),
                         _flat(free_stack, "free_stack", _I32, dev, (pages,)), _flat(free_count, "free_count", _I32, dev, (1,)), pages, _flat(work, "work", _U8, dev, (1,)),
                         work.numel(), _flat(status, "status", _I32, dev, (1,)), K._stream()), "smc_evict")
