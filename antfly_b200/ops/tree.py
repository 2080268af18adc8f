"""Speculation over trees of drafted tokens: the integer maps of a step, attention of a tree over the paged KV cache, and
the accept walk that keeps one path of it.

A tree of sequence b is ``parents[b]``: node i's parent is an earlier node (``parents[b, i] < i``) or -1 (a root).  Node 0 is
the sequence's last accepted token, the others are drafts.  A round is::

    masks, depths = tree_plan(parents)                                   # once for a fixed tree shape
    maps = step_maps(kv_before, q_lens, blocks, page, max_blocks, T, depths=depths)
    ...  every layer: K / V of the nodes go to maps.slots, then
    ctx = tree_attention(q, k, v, maps.block_tables, maps.q_starts, q_lens, maps.kv_lens, masks, q_lens, max_q_len)
    ...  the target picks a token at every node
    path, count, next_token = tree_accept(tokens, parents, target, caches=[(k_cache, v_cache, maps.slots.view(B, -1))])

after which the accepted nodes' rows are the first ``count`` of the tree and the sequence is truncated to
``kv_before + count``.  ``step_maps`` without ``depths`` serves every other packed step (prefill chunks, decode).

CUDA tensors run the kernels of ``csrc/kernels/tree_maps.cu`` and ``tree_attention.cu``; CPU tensors the plain forms of
:mod:`antfly_b200.ops.reference`.  Integer tensors are int32.  Lengths, links and block ids live on the device, so a value
that is out of range is not an exception: the kernels skip the access and set the status word that
:func:`antfly_b200._native.status` reads.  Calls run on the current stream of the tensors' device, which has to be the
calling thread's current device.
"""
from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import torch

from .. import _native as N
from . import reference as R
from .kv_quant import CodecLayer

MAX_NODES = 256       # nodes of one tree
MIN_SCALE, MAX_SCALE = 1e-7, 1e4     # of the scores of tree attention

_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_float


@functools.lru_cache(maxsize=None)
def _lib():
    lib = N.cuda()
    lib.afb_step_maps.argtypes = [_P, _P, _P, _I, _P, _L, _I, _P, _P, _I, _I, _I, _I, _P, _P, _P, _P, _P, _P, _P]
    lib.afb_tree_plan.argtypes = [_P, _L, _P, _I, _I, _P, _P, _P]
    lib.afb_tree_accept.argtypes = ([_P, _L] * 3 + [_P, _I, _I, _P, _P, _P] +
                                    [_P, _P, _L, _L, _I, _L, _P, _L, _I] * 2 + [_P])
    lib.afb_tree_attention.argtypes = [_P, _L, _P, _P, _I, _I, _I, _P, _L, _I, _P, _P, _P, _P, _P, _L, _I, _I, _P, _L, _P,
                                       _L, _I, _I, _I, _I, _I, _I, _I, _I, _I, _F, _P, _L, _P]
    lib.afb_tree_attention_scratch.argtypes = [_I] * 11
    lib.afb_tree_attention_scratch.restype = _L
    return lib


def _stream(*tensors) -> int:
    """The current stream's handle, once every tensor is on the thread's current device (the launchers' contract).  These
    operators are called once per layer and take a few microseconds on the device, so the handle is taken without
    building a ``torch.cuda.Stream``."""
    dev = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise N.NativeError(f"tensor on {t.device} passed to a kernel launcher while this thread's current device is "
                                f"cuda:{dev}; wrap the call in device_of(tensor.device)")
    return torch._C._cuda_getCurrentRawStream(dev)


_i32 = torch.int32
_INT_MAX = 2 ** 31 - 1
_CACHES = (torch.bfloat16, torch.float8_e4m3fn, torch.float32)


def _ints(name: str, t: torch.Tensor, *shape) -> torch.Tensor:
    """The tensor, int32 of that shape (None: any extent), with a contiguous last dimension."""
    if t.dtype is _i32 and t.shape == shape and t.is_contiguous():
        return t
    if t.dtype is not _i32 or t.dim() != len(shape) or any([w is not None and s != w for s, w in zip(t.shape, shape)]):
        want = ", ".join("*" if w is None else str(w) for w in shape)
        raise ValueError(f"{name} must be int32 [{want}], got {t.dtype} {list(t.shape)}")
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _row_stride(t: torch.Tensor, at: int, D: int) -> Optional[int]:
    """Elements between the tokens of [T, heads, D] if the kernels can take them as they lie (heads next to one another, rows
    that start on 16 bytes), else None."""
    tok, head, el = t.stride()
    return tok if el == 1 and head == D and tok % 8 == 0 and at % 16 == 0 else None


def _addr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


@dataclass
class StepMaps:
    """Integer inputs of a packed step.  ``positions`` / ``slots`` have ``num_tokens`` entries; those behind the last
    sequence's rows are 0 and -1 (a negative slot is not written to)."""
    q_starts: torch.Tensor       # [B] first packed row of each sequence
    kv_lens: torch.Tensor        # [B] keys with the step's own
    logit_rows: torch.Tensor     # [B] last packed row of each sequence
    positions: torch.Tensor      # [T]
    slots: torch.Tensor          # [T] block * page + offset
    block_tables: torch.Tensor   # [B, max_blocks], 0 behind a sequence's last block


def step_maps(kv_before: torch.Tensor, q_lens: torch.Tensor, blocks: torch.Tensor, page: int, max_blocks: int,
              num_tokens: int, depths: Optional[torch.Tensor] = None, tree_lens: Optional[torch.Tensor] = None,
              shift: Optional[torch.Tensor] = None) -> StepMaps:
    """Block tables, slots and positions of a step from the requests' lengths, in one launch.

    Sequence b has ``kv_before[b]`` keys in the cache and ``q_lens[b]`` rows in the step; ``blocks`` holds the block ids of
    all sequences one after another, ``ceil((kv_before[b] + q_lens[b]) / page)`` for sequence b.  ``num_tokens`` is the
    packed row count T (it may exceed the sum of ``q_lens``: a padded batch).  Row i of a sequence is key
    ``kv_before + i``, which is its position too; with ``depths`` [B, nodes] the rows are the last ``q_lens[b]`` of
    ``tree_lens[b]`` (default: ``q_lens``) tree nodes and sit at the first node's key plus their depth.  ``shift`` [B] is
    added to the positions (keys dropped from the cache, rotary offsets)."""
    B = q_lens.numel()
    q_lens, kv_before, blocks = _ints("q_lens", q_lens, B), _ints("kv_before", kv_before, B), _ints("blocks", blocks, blocks.numel())
    if tree_lens is not None:
        tree_lens = _ints("tree_lens", tree_lens, B)
    if shift is not None:
        shift = _ints("shift", shift, B)
    if depths is not None:
        depths = _ints("depths", depths, B, depths.shape[-1])
    if page < 1 or max_blocks < 0 or num_tokens < 0:
        raise ValueError(f"bad sizes: page {page}, max_blocks {max_blocks}, num_tokens {num_tokens}")
    if not q_lens.is_cuda:
        return StepMaps(*R.step_maps(kv_before, q_lens, blocks, page, max_blocks, num_tokens, depths, tree_lens, shift))
    stream = _stream(kv_before, q_lens, blocks, depths, tree_lens, shift)
    buf = torch.empty(3 * B + 2 * num_tokens + B * max_blocks, dtype=torch.int32, device=q_lens.device)
    tables, q_starts, kv_lens, rows, positions, slots = buf.split_with_sizes([B * max_blocks, B, B, B, num_tokens, num_tokens])
    if B == 0:
        positions.zero_()
        slots.fill_(-1)
    else:
        rc = _lib().afb_step_maps(
            kv_before.data_ptr(), q_lens.data_ptr(), blocks.data_ptr(), blocks.shape[0], _addr(depths),
            depths.stride(0) if depths is not None else 0, depths.shape[1] if depths is not None else 0,
            _addr(tree_lens), _addr(shift), B, page, max_blocks, num_tokens, q_starts.data_ptr(), kv_lens.data_ptr(),
            rows.data_ptr(), positions.data_ptr(), slots.data_ptr(), tables.data_ptr(), stream)
        N.check(rc, "afb_step_maps")
        N.count_launch()
    return StepMaps(q_starts, kv_lens, rows, positions, slots, tables.view(B, max_blocks))


def tree_plan(parents: torch.Tensor, lens: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """parents [B, nodes] (at most 256) -> (masks [B, nodes, ceil(nodes / 32)], depths [B, nodes]): bit j of node i's mask
    is set for i itself and every node on its way to a root; the depth counts the proper ancestors.  Nodes at ``lens[b]``
    and behind have no bits and depth 0.  A link that does not point to an earlier node is read as a root and reported
    through the status word."""
    B, nodes = parents.shape if parents.dim() == 2 else (None, None)
    parents = _ints("parents", parents, B, nodes)
    if not 1 <= nodes <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {nodes}")
    if lens is not None:
        lens = _ints("lens", lens, B)
    if not parents.is_cuda:
        return R.tree_plan(parents, lens)
    stream = _stream(parents, lens)
    masks = torch.empty((B, nodes, (nodes + 31) // 32), dtype=torch.int32, device=parents.device)
    depths = torch.empty((B, nodes), dtype=torch.int32, device=parents.device)
    rc = _lib().afb_tree_plan(parents.data_ptr(), parents.stride(0), _addr(lens), B, nodes, masks.data_ptr(),
                              depths.data_ptr(), stream)
    N.check(rc, "afb_tree_plan")
    N.count_launch()
    return masks, depths


def tree_attention(q, k_cache, v_cache, block_tables, q_starts, q_lens, kv_lens, masks, tree_lens, max_q_len: int,
                   max_kv: int = 0, scale: Optional[float] = None, window: int = 0,
                   depths: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of packed tree nodes q [T, Hq, D] (bf16) over the paged cache [num_blocks, page, Hkv, D] (bf16 or e4m3;
    a :class:`antfly_b200.ops.kv_quant.CodecLayer` too: fp8 as it lies, of the other codecs the pages of ``max_kv`` keys per
    sequence are expanded to bf16 in every call).  D is a multiple of 8 up to 256, Hq a multiple of Hkv.

    The last ``tree_lens[b]`` of sequence b's ``kv_lens[b]`` keys are its tree's nodes and its ``q_lens[b]`` rows the last of
    those nodes (all of them in a verification pass, one level of them while drafting).  A row sees every key in front
    of the tree and the nodes whose bit is set in its own mask row: ``masks`` [B, nodes, ceil(nodes / 32)] from
    :func:`tree_plan`, or any other; a batch dimension expanded from 1 serves one tree shape for all.  A row that sees
    no key comes back as zeros.  ``window`` > 0 (needs ``depths``) keeps the keys at positions > the row's position -
    ``window``, a node's position being the tree's first key plus its depth.  ``scale`` (default 1 / sqrt(D)) is a positive
    number from 1e-7 to 1e4; scaled scores lie below 2^30 in magnitude.

    Scores, their maxima, the sums of the weights and the output are kept in 32 bits.  For the product with V the GPU rounds
    each weight once to 16 bits (bf16; fp16 over e4m3 caches with many rows), and the output to bf16 in the end.

    ``max_q_len`` bounds ``q_lens`` and ``max_kv`` (0: what the block table can hold) bounds ``kv_lens``; both size the
    launch, and a length past them is reported through the status word.  A window of ``max_kv`` keys or more is none.
    The sequences' rows may lie in any order but do not overlap.  Rows of ``out`` that belong to no sequence are left as
    they were; in a new output they are zero."""
    if q.dim() != 3:
        raise ValueError(f"q must be [T, Hq, D], got {list(q.shape)}")
    T, Hq, D = q.shape
    B = q_lens.numel()
    q_starts, q_lens = _ints("q_starts", q_starts, B), _ints("q_lens", q_lens, B)
    kv_lens, tree_lens = _ints("kv_lens", kv_lens, B), _ints("tree_lens", tree_lens, B)
    block_tables = _ints("block_tables", block_tables, B, block_tables.shape[-1])
    if isinstance(k_cache, CodecLayer):
        if k_cache.codec == "fp8":
            shape = (k_cache.num_blocks, k_cache.page, k_cache.Hkv, D)
            k_cache, v_cache = (c.data.view(torch.float8_e4m3fn).view(shape) for c in (k_cache, v_cache))
        else:
            k_cache, v_cache, block_tables = _expanded(k_cache, v_cache, block_tables, kv_lens, max_kv)
    num_blocks, page, Hkv, Dk = k_cache.shape
    kind = k_cache.dtype
    if kind not in _CACHES or v_cache.dtype is not kind or v_cache.shape != k_cache.shape or Dk != D:
        raise ValueError(f"caches of one shape [blocks, page, Hkv, {D}] in bf16 or e4m3 are needed, got "
                         f"{k_cache.dtype} {list(k_cache.shape)} and {v_cache.dtype} {list(v_cache.shape)}")
    if D % 8 or not 8 <= D <= 256 or Hq % Hkv:
        raise ValueError(f"head width {D} (a multiple of 8 up to 256) or heads {Hq} over {Hkv} not supported")
    masks = _ints("masks", masks, B, *masks.shape[1:]) if masks.dim() == 3 else _ints("masks", masks, B, None, None)
    nodes = masks.shape[1]
    if not 1 <= nodes <= MAX_NODES or masks.shape[2] != (nodes + 31) // 32:
        raise ValueError(f"masks must be [B, nodes, ceil(nodes / 32)] with 1 to {MAX_NODES} nodes, got {list(masks.shape)}")
    if window > 0:
        if depths is None:
            raise ValueError("a sliding window needs the nodes' depths")
        depths = _ints("depths", depths, B, nodes)
    if max_q_len < 0 or max_kv < 0 or window < 0:
        raise ValueError("max_q_len, max_kv and window are not negative")
    if out is not None and (out.shape != q.shape or out.dtype != torch.bfloat16 or out.device != q.device):
        raise ValueError(f"out must be bf16 {list(q.shape)} on {q.device}")
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    if not MIN_SCALE <= scale <= MAX_SCALE:
        raise ValueError(f"scale must be a positive number from {MIN_SCALE:g} to {MAX_SCALE:g}, got {scale}")
    if not q.is_cuda:
        y = R.tree_attention(q, k_cache, v_cache, block_tables, q_starts, q_lens, kv_lens, masks, tree_lens, scale, window,
                             depths, out)
        return y if out is None else out.copy_(y)
    if q.dtype is not torch.bfloat16 or kind is torch.float32:
        raise NotImplementedError("tree attention reads bf16 queries and a bf16 or e4m3 cache")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("the caches must be contiguous")
    k_at, v_at, q_at = k_cache.data_ptr(), v_cache.data_ptr(), q.data_ptr()
    if (k_at | v_at) & 15:
        raise ValueError("the caches must be 16-byte aligned")
    if nodes > 1 and masks.stride(1) != masks.shape[2]:
        masks = masks.contiguous()
    stream = _stream(q, k_cache, v_cache, block_tables, q_starts, q_lens, kv_lens, masks, tree_lens, depths, out)
    row = _row_stride(q, q_at, D)
    if row is None:
        q = q.clone(memory_format=torch.contiguous_format)     # contiguous() would keep a base that is not aligned
        q_at, row = q.data_ptr(), Hq * D
    if out is None:
        y, y_row = torch.empty((T, Hq, D), dtype=torch.bfloat16, device=q.device), Hq * D
    else:
        y, y_row = out, _row_stride(out, out.data_ptr(), D)
        if y_row is None:
            y, y_row = out.clone(memory_format=torch.contiguous_format), Hq * D
    if B == 0:
        return y.zero_() if out is None else out
    # The keys of a sequence may be shared out over several CTAs, whose partial rows (32 bits) are joined in the end.
    reach = min(block_tables.shape[1] * page, max_kv or _INT_MAX, _INT_MAX)
    window, max_q_len = min(window, _INT_MAX), min(max_q_len, T, nodes)
    kv8 = 0 if kind is torch.bfloat16 else 1
    lib = _lib()
    floats = lib.afb_tree_attention_scratch(B, T, Hq, Hkv, D, kv8, page, nodes, window, max_q_len, reach)
    scratch = torch.empty(floats, dtype=torch.float32, device=q.device) if floats else None
    rc = lib.afb_tree_attention(
        q_at, row, k_at, v_at, kv8, num_blocks, page, block_tables.data_ptr(),
        block_tables.stride(0), block_tables.shape[1], q_starts.data_ptr(), q_lens.data_ptr(), kv_lens.data_ptr(),
        tree_lens.data_ptr(), masks.data_ptr(), masks.stride(0), nodes, masks.shape[2], _addr(depths),
        depths.stride(0) if depths is not None else 0, y.data_ptr(), y_row, B, T, Hq, Hkv, D, max_q_len, reach, window,
        1 if out is None else 0, scale, _addr(scratch), floats, stream)
    N.check(rc, "afb_tree_attention")
    N.count_launch(2 if floats else 1)
    return y if out is None or y is out else out.copy_(y)


def _expanded(k_cache, v_cache, block_tables, kv_lens, max_kv: int):
    """Caches kept in another codec: the pages that the step can see, expanded to bf16, with a block table of their own.  A
    block id that is none counts only where a key needs it."""
    page, Hkv, D = k_cache.page, k_cache.Hkv, k_cache.D
    nb = block_tables.shape[1]
    if max_kv > 0:
        nb = min(nb, (max_kv + page - 1) // page)
    B, dev = block_tables.shape[0], block_tables.device
    key = torch.arange(nb * page, device=dev)
    rows = (block_tables[:, :nb].long() * page)[:, :, None] + key[:page]
    rows = rows.view(B, -1).clamp(-1, k_cache.num_blocks * page)         # ids that are none stay so in 32 bits
    rows = torch.where(key < kv_lens[:, None], rows, 0).view(-1).int()
    kb, vb = (c.expand(rows).view(B * nb, page, Hkv, D) for c in (k_cache, v_cache))
    return kb, vb, torch.arange(B * nb, dtype=torch.int32, device=dev).view(B, nb)


def tree_accept(tokens: torch.Tensor, parents: torch.Tensor, target: torch.Tensor, lens: Optional[torch.Tensor] = None,
                caches: Sequence[tuple] = ()) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The accepted path of every tree: from node 0, the child (the lowest of several) whose token is what the target chose
    at the current node, until there is none.  ``tokens``, ``parents``, ``target`` [B, nodes]; ``lens`` [B] counts the
    nodes of a tree (default all, at least one).  Returns (path [B, nodes], -1 behind its end; count [B], the nodes on
    it with node 0; next_token [B], the target's choice at its last node).

    ``caches`` holds up to two ``(k, v, slots)`` or ``(k, v, slots, nodes)``: caches of all layers [L, num_blocks, page, ...]
    (or their :class:`antfly_b200.ops.kv_quant.CodecCache`) and the slots [B, nodes] of the nodes, of which only the first
    ``nodes`` were written (a draft model has no rows for its last level).  Row ``slots[b, path[i]]`` is moved to
    ``slots[b, i]`` in every layer; rows behind the path are left as they were.  The slots of all trees differ, and no two
    of the key and value tensors share memory."""
    B, nodes = tokens.shape if tokens.dim() == 2 else (None, None)
    tokens = _ints("tokens", tokens, B, nodes)
    parents, target = _ints("parents", parents, B, nodes), _ints("target", target, B, nodes)
    if not 1 <= nodes <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {nodes}")
    if lens is not None:
        lens = _ints("lens", lens, B)
    if len(caches) > 2:
        raise ValueError("at most two caches")
    rows, spans = [], []
    for k, v, slots, *held in caches:
        k, v = getattr(k, "data", k), getattr(v, "data", v)
        slots = _ints("slots", slots, B, nodes)
        if k.dim() < 4 or k.shape[:3] != v.shape[:3] or not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("caches must be contiguous [layers, blocks, page, ...]")
        rows.append((k, v, slots, held[0] if held else nodes))
        spans += (k.data_ptr(), k.nbytes), (v.data_ptr(), v.nbytes)
    for i, (a, n) in enumerate(spans):
        for b, m in spans[:i]:
            if a < b + m and b < a + n:
                raise ValueError("keys and values of the caches share memory: their rows would be moved twice")
    if not tokens.is_cuda:
        path, count, following = R.tree_accept(tokens, parents, target, lens)
        for k, v, slots, held in rows:
            R.keep_path(k, v, slots, path, held)
        return path, count, following
    stream = _stream(tokens, parents, target, lens, *(t for r in rows for t in r[:3]))
    buf = torch.empty(B * (nodes + 2), dtype=_i32, device=tokens.device)
    path, count, following = buf.split_with_sizes([B * nodes, B, B])
    path = path.view(B, nodes)
    args = []
    for i, (k, _, slots, held) in enumerate(rows):
        (k_at, k_bytes), (v_at, v_bytes) = spans[2 * i:2 * i + 2]
        layers, blocks, page = k.shape[:3]
        n = max(layers * blocks * page, 1)                   # (row sizes not from strides: a dimension of one has any)
        args += [k_at, v_at, k_bytes // n, v_bytes // n, layers, blocks * page, slots.data_ptr(), slots.stride(0), held]
    args += [0, 0, 0, 0, 0, 0, 0, 0, 0] * (2 - len(rows))
    rc = _lib().afb_tree_accept(tokens.data_ptr(), tokens.stride(0), parents.data_ptr(), parents.stride(0),
                                target.data_ptr(), target.stride(0), _addr(lens), B, nodes, path.data_ptr(),
                                count.data_ptr(), following.data_ptr(), *args, stream)
    N.check(rc, "afb_tree_accept")
    N.count_launch()
    return path, count, following
