"""Operators of language-model circuits: learning from a teacher's top logits, and answering with beams.

``top_logits`` takes the largest logits of a teacher's vocabulary rows, ``expected_log_probs`` scores tables of leaf
log-probabilities against them (and is what a compiled circuit computes at its leaves when it is called with a
:class:`TopLogits` instead of categories), ``beam_select`` picks the best continuations over beams and vocabulary and
``reorder`` moves the states of the beams along.  Everything runs in the CUDA library on torch's current stream of the
tensors' device; nothing synchronises, and every call can be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from typing import List, NamedTuple, Optional, Tuple

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib

MAX_TOP = 128                  # entries of one selection
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class TopLogits(NamedTuple):
    """What is kept of a teacher's distributions: the ids of a few categories per position and their logits.

    ``ids`` and ``logits`` have the same shape, slots last (for a circuit ``[B, num_vars, K]``); ids are int32 or int64,
    logits float32, bfloat16 or float16.  A slot is empty when its id is negative or its logit is -inf or NaN.  The weight
    of a slot is ``exp(logits / temperature - log_norm)``; without ``log_norm`` (the shape of ``ids`` less its last
    dimension), or where it is not finite, the weights of a position's slots sum to one.  A position whose slots are all
    empty says nothing: it is marginalised.  Logits of +inf share the whole weight of their position, with or without ``log_norm``.
    (A normaliser of 32 bits is exact to 2^-24 of its size: where logits go into the thousands, the weights' last digits go with it.)"""
    ids: torch.Tensor
    logits: torch.Tensor
    temperature: float = 1.0
    log_norm: Optional[torch.Tensor] = None

    def _check(self):
        if self.ids.dtype not in (torch.int32, torch.int64):
            raise TypeError("ids must be int32 or int64")
        if self.logits.dtype not in _TYPES:
            raise TypeError("logits must be float32, bfloat16 or float16")
        if self.ids.shape != self.logits.shape or self.ids.dim() < 1:
            raise ValueError(f"ids {tuple(self.ids.shape)} and logits {tuple(self.logits.shape)} must have the same shape")
        if not 0.0 < self.temperature < float("inf"):
            raise ValueError("`temperature` should be positive")
        if self.log_norm is not None and (self.log_norm.shape != self.ids.shape[:-1] or self.log_norm.dtype != torch.float32):
            raise ValueError("`log_norm` must be float32 with one value per position")


def _require_cuda(*tensors):
    device = tensors[0].device
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise NotImplementedError("language-model operators run on CUDA only (no CPU path)")
        if t is not None and t.device != device:
            raise ValueError(f"tensors on {device} and {t.device}")


def _refuse_tangents(name: str, *tensors):
    if getattr(forward_ad, "_current_level", 0) >= 0:            # (only within a level of forward-mode differentiation)
        if any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
            raise RuntimeError(f"`{name}` has no forward-mode derivative")


class _Geo(ctypes.Structure):
    """`PcxTeacherGeo` of the library: the leaf vectors that look at a teacher, and how wide it is."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("segs", "groups", "set_first", "set_vars")] + [("flow_cols", ctypes.c_int64)] + \
        [(n, ctypes.c_int32) for n in ("positions", "nodes", "cats", "tied", "n_segs", "n_groups", "n_sets", "max_vars",
                                       "total_vars", "width", "slots", "pad_")]


def _prepare(teacher: TopLogits, width: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Categories and weights of a teacher's slots, ``[T, width, K]`` pairs of 32 bits, from ids ``[B, T, K]``."""
    ids, x, norm = teacher.ids, teacher.logits, teacher.log_norm
    B, T, K = ids.shape
    if out is None:
        out = torch.empty(T, width, K, 2, dtype=torch.int32, device=ids.device)
    if out.numel() > 0:
        nb, nv = (0, 0) if norm is None else norm.stride()
        _lib.launch("pcx_teacher_prep", ids.device, out.data_ptr(), ids.data_ptr(), int(ids.dtype == torch.int64), *ids.stride(),
                    x.data_ptr(), _TYPES[x.dtype], *x.stride(), None if norm is None else norm.data_ptr(), nb, nv, B, T, K, width,
                    float(teacher.temperature))
    return out


class Entries:
    """A prepared batch of teacher's slots, in the place of a circuit's ``[V, W]`` categories."""
    __slots__ = ("tensor", "width", "slots")

    def __init__(self, tensor: torch.Tensor):
        self.tensor = tensor
        _, self.width, self.slots, _ = tensor.shape

    def data_ptr(self):
        """What a captured pass goes by: where the slots are, and how many."""
        return (self.tensor.data_ptr(), *self.tensor.shape)


def _form(named: int, C: int, M: int, own: bool) -> int:
    """How the forward pass reads tables of M nodes and C categories that ``named`` slots each look up (``own``: the table
    belongs to one position).  2, through shared memory, takes the whole table once: tables of one position, at least an
    eighth of whose categories are named, as long as 64 of their nodes fit (196 tables of 256 x 256, batch 100, 16 slots:
    47 us, 62 turned, 387 in place; 64 of 512 x 1000, batch 77: 86, 68, 209).  3, turned, writes and reads the table once more
    but then finds the nodes of a category side by side: from a quarter of the categories on.  0, in place, touches a sector
    of 32 bytes per slot and node."""
    if own and M > 1 and named * 8 >= C and _lib.load().pcx_teacher_staged_nodes(C, M) >= min(64, M):
        return 2
    return 3 if M > 1 and named * 4 >= C else 0


class LeafTables:
    """The leaf vectors of an input layer as the teacher's kernels walk them: vectors, groups that share a table (in the
    order of their first vector), and the variables of each group."""

    def __init__(self, vectors, num_params: int, device):
        """``vectors``: (variable, nodes, categories, first row of the value buffers, first parameter, first flow or None for a
        tied vector) of every leaf vector; ``num_params``: parameters of all of them."""
        cats = {v[2] for v in vectors}
        cats_per_row = min(cats) if len(cats) == 1 else 0           # (tables can be turned as one)
        self.rows = num_params // cats_per_row if cats_per_row else 0
        segs, groups, sets, by_table = [], [], {}, {}
        for v in vectors:
            by_table.setdefault(v[4], []).append(v)
        flow_col = 0
        for table, members in by_table.items():
            M, C = members[0][1:3]
            col = table // cats_per_row if cats_per_row else 0
            at = sets.setdefault(tuple(v[0] for v in members), len(sets))
            groups.append((at, M, C, col, next(v[5] for v in members if v[5] is not None), flow_col))
            for var, _, _, row0, _, _ in members:
                segs.append((var, M, C, col, row0, table, flow_col))
                flow_col += -(-M // 4) * 4
        self.cols_by_four = all(s[3] % 4 == 0 for s in segs)
        seg = np.zeros(len(segs), dtype=[("a", np.int32, 4), ("b", np.int64, 3)])
        seg["a"], seg["b"] = [s[:4] for s in segs], [s[4:] for s in segs]
        grp = np.zeros(len(groups), dtype=[("a", np.int32, 4), ("b", np.int64, 2)])
        grp["a"], grp["b"] = [g[:4] for g in groups], [g[4:] for g in groups]
        first = np.cumsum([0] + [len(v) for v in sets]).astype(np.int32)
        on = lambda a: torch.from_numpy(a.view(np.uint8).copy()).to(device)
        self._held = [on(seg), on(grp), on(first), on(np.concatenate([np.asarray(v, np.int32) for v in sets]))]
        self.sizes = dict(flow_cols=flow_col, nodes=max(s[1] for s in segs), cats=max(s[2] for s in segs), n_segs=len(segs),
                          n_groups=len(groups), n_sets=len(sets), max_vars=max(len(v) for v in sets), total_vars=int(first[-1]))

    def geo(self, entries: Entries) -> _Geo:
        return _Geo(*[t.data_ptr() for t in self._held], width=entries.width, slots=entries.slots, **self.sizes)

    def _named(self, entries: Entries) -> int:
        """Slots that look one table up."""
        return self.sizes["max_vars"] * entries.width * entries.slots

    def forward(self, node_mars: torch.Tensor, params: torch.Tensor, entries: Entries, turned_stride: int = 0):
        """``params``: probabilities of the tables, or (``turned_stride``) their transposed logarithms."""
        geo, take_log = self.geo(entries), 1
        form = 3 if turned_stride else _form(self._named(entries), geo.cats, geo.nodes, geo.max_vars == 1)
        if form == 3 and not turned_stride:
            if 0 < self.rows < 2 ** 29:
                turned_stride = -(-self.rows // 4) * 4
                turned = torch.empty(geo.cats, turned_stride, dtype=torch.float32, device=params.device)
                _lib.call("pcx_teacher_turn", turned, params, self.rows, geo.cats, turned_stride, 1)
                params = turned
            else:
                form = 0
        if form == 3:
            take_log = 0
            form = 3 if self.cols_by_four and turned_stride % 4 == 0 else 1
        _lib.call("pcx_teacher_fwd", node_mars, params, entries.tensor, ctypes.addressof(geo), form, turned_stride, take_log)

    def backward(self, flows: torch.Tensor, node_flows: torch.Tensor, entries: Entries, logspace: bool, turned_stride: int = 0,
                 touched: Optional[torch.Tensor] = None):
        """Adds to the accumulators of the tables, or (``turned_stride``) to transposed ones."""
        geo = self.geo(entries)
        runs = int(self._named(entries) * 16 < geo.cats)
        scratch = torch.empty(_lib.load().pcx_teacher_bwd_scratch_bytes(ctypes.addressof(geo), runs), dtype=torch.uint8,
                              device=flows.device)
        _lib.call("pcx_teacher_bwd", flows, touched, scratch, node_flows, entries.tensor, ctypes.addressof(geo),
                  2 if turned_stride else 1, runs, turned_stride, int(logspace))


@functools.lru_cache(maxsize=256)
def _sizes(T: int, M: int, C: int, W: int, K: int, tied: bool):
    """(`_Geo` of T positions of M nodes, its address, form of the forward pass, row width of the turned table, whether the
    backward pass visits only categories that occur, bytes of its workspace)."""
    n, lib = (1 if tied else T), _lib.load()
    geo = _Geo(flow_cols=T * -(-M // 4) * 4, positions=T, nodes=M, cats=C, tied=int(tied), n_segs=T, n_groups=n, n_sets=n,
               max_vars=T if tied else 1, total_vars=T, width=W, slots=K)
    named = geo.max_vars * W * K                        # slots that look a table up
    form, stride = _form(named, C, M, not tied), 0
    if form == 3:                                       # (rows of a turned table are addressed with 32 bits)
        stride = -(-(n * M) // 4) * 4 if n * M < 2 ** 29 else 0
        form = 0 if stride == 0 else 3 if tied or M % 4 == 0 else 1
    runs = int(named * 16 < C)
    at = ctypes.addressof(geo)
    return geo, at, form, stride, runs, lib.pcx_teacher_bwd_scratch_bytes(at, runs)


def _expect(log_probs, teacher):
    """Values and the prepared slots of the teacher."""
    ids, x, norm, device = teacher.ids, teacher.logits, teacher.log_norm, log_probs.device
    B, T, K = ids.shape
    M, C = log_probs.shape[-2:]
    entries = torch.empty(T, B, K, 2, dtype=torch.int32, device=device)
    out = torch.empty(T, M, B, dtype=torch.float32, device=device)
    if T * M * B * K == 0:
        return out.zero_(), entries
    plan = _sizes(T, M, C, B, K, log_probs.dim() == 2)  # (holds what `geo` is the address of)
    geo, form, stride = plan[1:4]
    table = log_probs.contiguous()
    turned = torch.empty(C, stride, dtype=torch.float32, device=device) if stride else None
    nb, nv = (0, 0) if norm is None else norm.stride()
    _lib.launch("pcx_teacher_expect", device, out.data_ptr(), entries.data_ptr(), None if turned is None else turned.data_ptr(),
                table.data_ptr(), ids.data_ptr(), int(ids.dtype == torch.int64), *ids.stride(), x.data_ptr(), _TYPES[x.dtype],
                *x.stride(), None if norm is None else norm.data_ptr(), nb, nv, B, float(teacher.temperature), geo, form, stride)
    return out, entries


class _Expected(torch.autograd.Function):
    """Values of leaf tables under a teacher; the gradient of the tables."""

    @staticmethod
    def forward(ctx, log_probs, teacher):
        out, ctx.entries = _expect(log_probs, teacher)  # (neither an input's memory nor an output's)
        ctx.shape = log_probs.shape
        return out

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled() and grad.requires_grad:
            raise RuntimeError("`expected_log_probs` is differentiable once")
        entries, shape = ctx.entries, ctx.shape
        T, W, K, _ = entries.shape
        device = entries.device
        if grad.numel() == 0 or K == 0:
            return torch.zeros(shape, dtype=torch.float32, device=device), None
        plan = _sizes(T, shape[-2], shape[-1], W, K, len(shape) == 2)
        out = torch.empty(*shape, dtype=torch.float32, device=device)
        scratch = torch.empty(plan[5], dtype=torch.uint8, device=device)
        grad = grad.contiguous()
        _lib.launch("pcx_teacher_bwd", device, out.data_ptr(), None, scratch.data_ptr(), grad.data_ptr(), entries.data_ptr(),
                    plan[1], 0, plan[4], 0, 0)
        return out, None


def expected_log_probs(log_probs: torch.Tensor, teacher: TopLogits) -> torch.Tensor:
    """Log-probabilities of leaf tables expected under a teacher: ``out[t, m, b] = sum_k w[b, t, k] * log_probs[t, m, ids[b, t,
    k]]`` with the weights of ``teacher`` (see :class:`TopLogits`), whose ids are ``[B, T, K]``.

    ``log_probs`` (float32) is ``[M, C]``, one table of M nodes for all T positions, or ``[T, M, C]``, a table for each.
    Empty slots add nothing, whatever they hold; a weight of zero takes nothing of a log-probability of -inf; an id of C
    or more has the log-probability -inf.  Returns float32 ``[T, M, B]``.  The gradient goes to ``log_probs`` (sums in a
    fixed order: the same bits on every call), none to the teacher; second and forward-mode derivatives are refused.  Up
    to a million categories, 2^30 slots that share a table, 2^31 nodes over all positions.  A backward pass captured into a CUDA
    graph needs, as torch's own do, that no eager graph of the same leaf is alive while it is captured.

    Where a table's slots name a quarter of its categories or more, the call makes a turned copy of the tables, as large as they are."""
    teacher._check()
    if log_probs.dtype != torch.float32 or log_probs.dim() not in (2, 3):
        raise TypeError("log_probs must be float32 [M, C] or [T, M, C]")
    if teacher.ids.dim() != 3:
        raise ValueError("the teacher's ids must be [B, T, K]")
    B, T, K = teacher.ids.shape
    if log_probs.dim() == 3 and log_probs.size(0) != T:
        raise ValueError(f"{log_probs.size(0)} tables for {T} positions")
    if not 1 <= log_probs.size(-1) <= 1000000:
        raise ValueError("tables of 1 to 1000000 categories are supported")
    if max(B * K, 1) * (T if log_probs.dim() == 2 else 1) >= 2 ** 30:
        raise ValueError("more than 2^30 slots share a table")
    if T * log_probs.size(-2) >= 2 ** 31 or log_probs.size(-2) > 2 ** 30 - 4:         # (rows of flows are addressed with 32 bits)
        raise ValueError("more than 2^31 nodes over all positions, or 2^30 of one")
    _refuse_tangents("expected_log_probs", log_probs)
    _require_cuda(log_probs, teacher.ids, teacher.logits, teacher.log_norm)
    if log_probs.requires_grad and torch.is_grad_enabled():
        return _Expected.apply(log_probs, teacher)
    return _expect(log_probs.detach() if log_probs.requires_grad else log_probs, teacher)[0]


@functools.lru_cache(maxsize=None)
def _sm_count(index: int) -> int:
    return torch.cuda.get_device_properties(index).multi_processor_count


def _scratch(rows: int, row_bytes: int, n: int, device) -> Tuple[torch.Tensor, int]:
    """Workspace of a selection, and how its rows are walked: 0 for a warp a row, else the parts that a row is cut into.

    A warp a row keeps sixteen rows in flight per SM, without barriers, and costs short rows no idle threads.  Fewer and longer
    rows go to CTAs, four per SM if the rows give as many parts of 8 KB.  Calls of a warp a row against a CTA a row, us: 8192 rows of
    64 KB bf16, n = 32: 190, 231; 1024 of them: 36 both; 1776 of 16, 64, 196, 512 KB: n = 32: 30, 38; 56, 68; 144, 139; 298, 276;
    n = 128: 122, 227; 109, 351; 254, 485; 450, 687; the same in fp32: n = 32: 18, 32; 33, 52; 90, 111; 183, 218.  Long lists of fewer
    rows would be better off with a warp too, which the rule leaves out (1024 rows of 196 KB bf16, n = 128: 204, 308; 1001 of fp32, n =
    100: 96, 107)."""
    sms = _sm_count(device.index)
    splits = 0 if rows >= sms * 12 or row_bytes <= 8192 else max(1, min(-(-sms * 4 // rows), -(-row_bytes // 8192), 32))
    return torch.empty(rows * (max(splits, 1) + 1) * (8 * n + 16), dtype=torch.uint8, device=device), splits


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0) -> TopLogits:
    """The ``k`` largest logits of every row of ``logits`` ``[..., V]``, largest first, a lower id first among equals, and
    the rows' log-normalisers ``log sum_v exp(logits[v] / temperature)``.

    Returns a :class:`TopLogits` of ids (int64) and logits (in the type of the input) ``[..., k]`` and ``log_norm``
    ``[...]`` (float32).  Logits of -inf and NaN are no candidates and count nothing; a slot without a candidate has the id
    -1 and the logit -inf.  No gradient passes.  ``k`` is at most 128."""
    if logits.dtype not in _TYPES:
        raise TypeError("logits must be float32, bfloat16 or float16")
    if logits.dim() < 1 or not 1 <= logits.size(-1) < 2 ** 30:
        raise ValueError("logits need a vocabulary in their last dimension")
    V, lead = logits.size(-1), logits.shape[:-1]
    if not 1 <= k <= min(MAX_TOP, V):
        raise ValueError(f"`k` should be in [1, {min(MAX_TOP, V)}], got {k}")
    if not 0.0 < temperature < float("inf"):
        raise ValueError("`temperature` should be positive")
    _require_cuda(logits)
    x = logits
    if x.dim() != 2 or x.stride(1) != 1:
        x = x.detach().reshape(-1, V)
        x = x if x.stride(1) == 1 or V == 1 else x.contiguous()
    rows, device = x.size(0), x.device
    ids = torch.empty(*lead, k, dtype=torch.int64, device=device)       # (sizes one by one: a tuple of them costs a microsecond)
    values = torch.empty(*lead, k, dtype=x.dtype, device=device)
    norms = torch.empty(*(lead or ((),)), dtype=torch.float32, device=device)
    if rows > 0:
        scratch, splits = _scratch(rows, V * x.element_size(), k, device)
        _lib.launch("pcx_top_logits", device, ids.data_ptr(), values.data_ptr(), norms.data_ptr(), scratch.data_ptr(), x.data_ptr(),
                    _TYPES[x.dtype], rows, V, x.stride(0), k, splits, float(temperature))
    return TopLogits(ids, values, temperature, norms)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, num_out: Optional[int] = None,
                finished: Optional[torch.Tensor] = None, pad_id: int = 0, normalize: bool = True):
    """The ``num_out`` best continuations of every sequence's beams.

    ``logits`` ``[B, K, V]`` over the vocabulary, ``scores`` ``[B, K]`` (float32) of the beams so far.  Continuing beam k
    with token v scores ``scores[k] + logits[k, v] - logsumexp(logits[k])`` (``normalize=False``: the logits are
    log-probabilities already and are added as they are).  Sums are compared in 64 bits, larger first, a lower
    ``k * V + v`` first among equals.  A beam whose score is -inf or NaN is dead; logits of -inf or NaN are no
    continuations, and a row that holds +inf has none under ``normalize``.  A beam marked in ``finished`` (bool ``[B, K]``)
    has one continuation, ``pad_id`` at its own score.

    Returns scores (float32), parent beams and tokens (int64), each ``[B, num_out]``, best first; where there are fewer
    continuations the rest has the score -inf, parent 0 and token -1.  ``num_out`` defaults to K and is at most 128.  Not
    differentiable."""
    if logits.dtype not in _TYPES:
        raise TypeError("logits must be float32, bfloat16 or float16")
    if logits.dim() != 3:
        raise ValueError("logits must be [B, K, V]")
    B, K, V = logits.shape
    if scores.shape != (B, K) or scores.dtype != torch.float32:
        raise ValueError("scores must be float32 [B, K]")
    if finished is not None and (finished.shape != (B, K) or finished.dtype != torch.bool):
        raise ValueError("`finished` must be bool [B, K]")
    if not 1 <= K <= MAX_TOP or V < 1 or K * V >= 2 ** 31:
        raise ValueError(f"1 to {MAX_TOP} beams over a vocabulary with K * V < 2^31 are supported")
    n = K if num_out is None else int(num_out)
    if not 1 <= n <= min(MAX_TOP, K * V):
        raise ValueError(f"`num_out` should be in [1, {min(MAX_TOP, K * V)}], got {n}")
    if not 0 <= pad_id < V:
        raise ValueError("`pad_id` is not in the vocabulary")
    _require_cuda(logits, scores, finished)
    x = logits if logits.stride(2) == 1 or V == 1 else logits.detach().contiguous()
    scores = scores if scores.is_contiguous() else scores.detach().contiguous()
    finished = None if finished is None else finished.contiguous()
    device = x.device
    out = torch.empty(B, n, dtype=torch.float32, device=device)
    parents = torch.empty(B, n, dtype=torch.int64, device=device)
    tokens = torch.empty(B, n, dtype=torch.int64, device=device)
    if B > 0:
        scratch, splits = _scratch(B * K, V * x.element_size(), n, device)
        _lib.launch("pcx_beam_select", device, out.data_ptr(), parents.data_ptr(), tokens.data_ptr(), scratch.data_ptr(), x.data_ptr(),
                    _TYPES[x.dtype], scores.data_ptr(), None if finished is None else finished.data_ptr(), B, K, V, x.stride(0),
                    x.stride(1), n, pad_id, int(bool(normalize)), splits)
    return out, parents, tokens


def _beam_rows(x: torch.Tensor, dim: int):
    """(tensor, outer rows, bytes per beam, strides in bytes of outer rows and beams) of a state as the kernel walks it: a
    copy where the dimensions before or after the beams are not laid out as one."""
    size, es = x.shape, x.element_size()
    if x.is_contiguous():
        inner = math.prod(size[dim + 1:]) * es
        return x, math.prod(size[:dim]), inner, inner * size[dim], inner
    stride, inner = x.stride(), 1
    for d in range(x.dim() - 1, dim, -1):
        if size[d] != 1 and stride[d] != inner:
            return _beam_rows(x.contiguous(), dim)
        inner *= size[d]
    outer, step = 1, 0
    for d in range(dim - 1, -1, -1):
        if size[d] != 1:
            if outer == 1:
                step = stride[d]
            elif stride[d] != step * outer:
                return _beam_rows(x.contiguous(), dim)
            outer *= size[d]
    return x, outer, inner * es, step * es, stride[dim] * es


def reorder(parents: torch.Tensor, *states: torch.Tensor, dim: int = 0) -> List[torch.Tensor]:
    """The states of the beams that were continued: ``parents`` ``[B, n]`` (int32 or int64) names, for every new beam of a
    sequence, the old beam it continues; every state has B * K beams in dimension ``dim``, those of a sequence together.

    Returns the new states, contiguous, with B * n beams in that dimension.  A parent outside [0, K) gives zeros.  States
    may have any real type, other shapes than each other, and any strides; they are not differentiable."""
    wide = parents.dtype == torch.int64
    if parents.dim() != 2 or not (wide or parents.dtype == torch.int32):
        raise ValueError("`parents` must be int32 or int64 [B, n]")
    B, n = parents.shape
    moved, beams = [], None
    for x in states:
        size = x.shape
        if not -len(size) <= dim < len(size):
            raise ValueError(f"a state of shape {tuple(size)} has no dimension {dim}")
        at = dim % len(size)
        if x.is_complex():
            raise TypeError("states must be real")
        if x.requires_grad and torch.is_grad_enabled():
            raise ValueError("`reorder` is not differentiable: call it under torch.no_grad()")
        width = size[at]
        if B > 0 and (width == 0 or width % B != 0 or (beams is not None and width != B * beams)):
            raise ValueError(f"a state with {width} beams does not fit {B} sequences" +
                             (f" of {beams}" if beams is not None else ""))
        beams = width // B if B > 0 else 1
        moved.append((x, at, size))
    _refuse_tangents("reorder", *states)
    _require_cuda(parents, *states)
    parents, device = parents.contiguous(), parents.device
    out, held, rows = [], [], []
    for x, at, size in moved:
        x, outer, nbytes, outer_step, beam_step = _beam_rows(x, at)
        y = torch.empty(*size[:at], B * n, *size[at + 1:], dtype=x.dtype, device=device)
        out.append(y)
        if outer * nbytes * B * n > 0:
            source = x.data_ptr()
            bits = source | nbytes | outer_step | beam_step | 16
            held.append(x)                              # (a copy has to live until the launch)
            rows += (source, y.data_ptr(), outer, nbytes, outer_step, beam_step, bits & -bits)
    for i in range(0, len(rows), 56):
        part = rows[i:i + 56]
        _lib.launch("pcx_reorder", device, struct.pack(f"{len(part)}q", *part), len(part) // 7, parents.data_ptr(), int(wide), B,
                    beams, n)
    return out
