"""Word logits [N, V] (the speaker's vocabulary head): what shapes them before a word is drawn, and what a student learns from a teacher's.

    constrain_logits   penalties for repeated words, word biases, grammar masks          (differentiable; in place for decoding)
    top_logits         the k largest logits of every row and the log-mass of the others  (a teacher's targets; k = 1: the greedy word)
    distill_loss       the loss of a student against such targets, with its gradient     (differentiable)

fp32 or bf16 logits, rows any distance apart; arithmetic in fp32, one rounding to the logits' type at the end.  There is no CPU
fallback.  Everything is launched on the current stream of the logits' device; nothing synchronises, nothing is kept between calls."""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Optional, Union

import torch

from . import _lib, losses, ops

_p = ops._p
_TYPES = {torch.float32: ops.F32, torch.bfloat16: ops.BF16}


def _on(device):
    """The launches go to the logits' device, also when another one is current."""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _rows(t: torch.Tensor, name: str):
    """[N, V] word logits of a supported type, as rows of contiguous elements."""
    losses._not_deferred(t, name)
    if t.dtype not in _TYPES:
        raise TypeError(f"{name}: expected float32 or bfloat16 logits, got {t.dtype}")
    if t.dim() != 2 or t.shape[1] < 1 or t.shape[0] >= 1 << 31 or t.shape[1] >= 1 << 31:
        raise ValueError(f"{name}: expected logits [N, V] with V >= 1, got {tuple(t.shape)}")


def _gpu(t: torch.Tensor, name: str):
    if not t.is_cuda:
        raise _lib.VlnError(f"{name}: expected GPU tensors (the HIP path has no CPU fallback)")


def _dense(t: torch.Tensor):
    """`t` if its rows are contiguous and do not overlap, else a copy that is such."""
    return t if t.shape[1] == 1 or t.stride(1) == 1 and (t.shape[0] == 1 or t.stride(0) >= t.shape[1]) else t.contiguous()


def _ld(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]


def _list(t, N: int, device, dtype, name: str, shared: bool = False):
    """A per-row list [N, n] (shared: also [n], the same for every row) on the logits' device, its last dimension contiguous."""
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name}: on {t.device}, the logits are on {device}")
    if shared and t.dim() == 1:
        t = t.unsqueeze(0).expand(N, -1)
    if t.dim() != 2 or t.shape[0] != N:
        raise ValueError(f"{name}: expected [{N}, n], got {tuple(t.shape)}")
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _vector(t, N: int, device, dtype, name: str):
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name}: on {t.device}, the logits are on {device}")
    if tuple(t.shape) != (N,):
        raise ValueError(f"{name}: expected [{N}], got {tuple(t.shape)}")
    return t.detach().contiguous()


# ---- constraints -----------------------------------------------------------------------------------------------------------------
def pack_allowed(mask: torch.Tensor) -> torch.Tensor:
    """bool [G, V] (True = the word is allowed) -> int32 [G, ceil(V / 32)], word v at bit v % 32 of element v // 32: the mask rows that
    constrain_logits reads.  For a grammar's states, packed once; runs wherever the mask lives."""
    if mask.dtype != torch.bool or mask.dim() != 2:
        raise TypeError("pack_allowed: expected a bool mask [G, V]")
    G, V = mask.shape
    words = (V + 31) // 32
    bits = torch.zeros(G, words * 32, dtype=torch.int64, device=mask.device)
    bits[:, :V] = mask.to(torch.int64)
    packed = (bits.view(G, words, 32) << torch.arange(32, device=mask.device)).sum(2)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)


def _constrain_call(src, dst, logits, lists, backward: bool):
    a = _lib.Constrain()
    setattr(a, "in", src.data_ptr())
    a.out, a.ld_in, a.ld_out = dst.data_ptr(), _ld(src), _ld(dst)
    if backward:
        a.logits, a.ld_logits = logits.data_ptr(), _ld(logits)
    for k, v in lists["fields"].items():
        setattr(a, k, v.data_ptr() if torch.is_tensor(v) else v)
    a.type, (a.B, a.V), a.backward = _TYPES[src.dtype], src.shape, int(backward)
    _lib.check(_lib.load().vln_constrain_logits(C.byref(a), _lib.raw_stream()), "vln_constrain_logits")


class _Constrain(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, lists):
        z = _dense(logits.detach())
        out = torch.empty(z.shape, dtype=z.dtype, device=z.device)
        with _on(z.device):
            _constrain_call(z, out, None, lists, False)
        ctx.save_for_backward(logits, *lists["tensors"])         # (a list changed in place before the backward is an error, not a wrong gradient)
        ctx.lists = lists
        return out

    @staticmethod
    def backward(ctx, dout):
        z = _dense(ctx.saved_tensors[0].detach())
        d = _dense(dout.detach())
        dz = torch.empty(z.shape, dtype=z.dtype, device=z.device)
        with _on(z.device):
            _constrain_call(d, dz, z, ctx.lists, True)
        return dz, None


def constrain_logits(logits: torch.Tensor, *, history: Optional[torch.Tensor] = None, history_lengths: Optional[torch.Tensor] = None,
                     prompt: Optional[torch.Tensor] = None, prompt_lengths: Optional[torch.Tensor] = None,
                     repetition: Union[float, torch.Tensor] = 1.0, presence: Union[float, torch.Tensor] = 0.0,
                     frequency: Union[float, torch.Tensor] = 0.0, bias_ids: Optional[torch.Tensor] = None,
                     bias_values: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None,
                     allowed_rows: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Word logits [N, V] under constraints, in one launch (the reference only bans <UNK>, speaker.py:336):

        t = z;  words in `history` or `prompt`:  t = t / repetition if t > 0 else t * repetition
        words in `history`:                      t -= frequency * (times in history) + presence
        t += the word's `bias_values`;  words that `allowed` bans: -inf

    history [N, H] / prompt [N, P]: int64 word ids, any row stride (a slice of the words so far), valid up to *_lengths [N] int64 (None:
    all); ids outside [0, V) -- padding: -1 -- stand for no word.  repetition (> 0) / presence / frequency: a number, or float32 [N].
    bias_ids int64 / bias_values float32: [N, n] or [n] for every row, n <= 2048; a word listed twice gets both.  allowed: int32 mask
    rows [G, ceil(V / 32)] from `pack_allowed`; allowed_rows int64 [N] picks each row's (-1: unconstrained; anything else outside [0, G)
    bans every word, which is visible, never a read out of range); without it G is N, or 1 for all.  A row whose mask allows nothing is
    -inf throughout.

    out: where to write (same shape and type; `logits` itself: in place, untouched words are not even read).  Without `out` the result
    carries gradients to `logits` (0 for banned words); penalties and biases are constants."""
    _rows(logits, "constrain_logits")
    N, V = logits.shape
    dev = logits.device
    fields, tensors = {}, []

    def put(name, t):
        fields[name] = t
        tensors.append(t)

    for name, size, ids, lens in (("history", "H", history, history_lengths), ("prompt", "P", prompt, prompt_lengths)):
        if ids is None:
            if lens is not None:
                raise ValueError(f"constrain_logits: {name}_lengths without {name}")
            continue
        t = _list(ids, N, dev, torch.int64, f"constrain_logits: {name}")
        if t.shape[1] >= 1 << 31:
            raise ValueError(f"constrain_logits: {name} is longer than 2^31 words")
        if t.shape[1]:
            put(name, t)
            fields[size], fields["ld_" + name] = t.shape[1], t.stride(0)
            if lens is not None:
                put(name + "_len", _vector(lens, N, dev, torch.int64, f"constrain_logits: {name}_lengths"))
    for name, v, low in (("repetition", repetition, 0.0), ("presence", presence, None), ("frequency", frequency, None)):
        if torch.is_tensor(v):
            if v.requires_grad and torch.is_grad_enabled():
                raise ValueError(f"constrain_logits: {name} is a constant, it gets no gradient (detach it)")
            put(name, _vector(v, N, dev, torch.float32, f"constrain_logits: {name}"))
        else:
            v = float(v)
            if v != v or abs(v) == float("inf") or low is not None and v <= low:
                raise ValueError(f"constrain_logits: {name} = {v}")
            fields[name + "_all"] = v
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("constrain_logits: bias_ids and bias_values belong together")
    if bias_ids is not None:
        if bias_values.requires_grad and torch.is_grad_enabled():
            raise ValueError("constrain_logits: bias_values are constants, they get no gradient (detach them)")
        bi = _list(bias_ids, N, dev, torch.int64, "constrain_logits: bias_ids", True)
        bv = _list(bias_values.detach(), N, dev, torch.float32, "constrain_logits: bias_values", True)
        if bi.shape != bv.shape or bi.shape[1] > _lib.CONSTRAIN_MAX_BIAS:
            raise ValueError(f"constrain_logits: bias_ids {tuple(bias_ids.shape)} and bias_values {tuple(bias_values.shape)} must match, "
                             f"at most {_lib.CONSTRAIN_MAX_BIAS} per row")
        if bi.shape[1]:
            put("bias_ids", bi)
            put("bias_values", bv)
            fields["n_bias"], fields["ld_bias_ids"], fields["ld_bias_values"] = bi.shape[1], bi.stride(0), bv.stride(0)
    if allowed is None:
        if allowed_rows is not None:
            raise ValueError("constrain_logits: allowed_rows without allowed")
    else:
        if allowed.dim() != 2 or allowed.shape[0] < 1 or allowed.shape[1] != (V + 31) // 32:
            raise ValueError(f"constrain_logits: allowed must be [G >= 1, {(V + 31) // 32}] for {V} words, got {tuple(allowed.shape)}")
        al = _dense(_list(allowed, allowed.shape[0], dev, torch.int32, "constrain_logits: allowed"))
        if allowed_rows is None and al.shape[0] not in (1, N):
            raise ValueError(f"constrain_logits: {al.shape[0]} mask rows for {N} rows of logits need allowed_rows")
        put("allowed", al)
        fields["G"], fields["ld_allowed"] = al.shape[0], _ld(al)
        if allowed_rows is not None:
            put("allowed_rows", _vector(allowed_rows, N, dev, torch.int64, "constrain_logits: allowed_rows"))
    lists = {"fields": fields, "tensors": tensors}
    if out is None:
        _gpu(logits, "constrain_logits")
        if N == 0:
            return logits.clone()
        return _Constrain.apply(logits, lists)
    if logits.requires_grad and torch.is_grad_enabled() or out.requires_grad:
        raise ValueError("constrain_logits: out= carries no gradient; leave it out, or call it under torch.no_grad() on detached logits")
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev:
        raise ValueError(f"constrain_logits: out must be {tuple(logits.shape)} {logits.dtype} on {dev}")
    for t, name in ((logits, "logits"), (out, "out")):
        if N and _dense(t) is not t:
            raise ValueError(f"constrain_logits: with out=, the rows of {name} must be contiguous and must not overlap")
    if out.data_ptr() != logits.data_ptr() or _ld(out) != _ld(logits):
        lo = lambda t: t.data_ptr()
        hi = lambda t: t.data_ptr() + ((N - 1) * _ld(t) + V) * t.element_size()
        if N and lo(out) < hi(logits) and lo(logits) < hi(out):
            raise ValueError("constrain_logits: out overlaps the logits without being the same tensor")
    _gpu(logits, "constrain_logits")
    if N:
        with _on(dev):
            _constrain_call(logits.detach(), out, None, lists, False)
    return out


# ---- a teacher's top logits ------------------------------------------------------------------------------------------------------
def _temperature(T, who):
    T = float(T)
    if not _lib.TEMPERATURE_MIN <= T <= _lib.TEMPERATURE_MAX:
        raise ValueError(f"{who}: temperature {T} outside [{_lib.TEMPERATURE_MIN}, {_lib.TEMPERATURE_MAX}]")
    return T


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0):
    """(values [N, k], ids [N, k] int64, rest [N] float32): the k largest logits of every row, largest first, equal ones in the order of
    their ids (NaN counts as largest), and `rest = logsumexp(all other logits / temperature)` (-inf: none) -- the targets that
    `distill_loss` takes; `ids` with k = 1 is the greedy word.  1 <= k <= min(V, 256).  No gradient: a teacher is a constant."""
    _rows(logits, "top_logits")
    T = _temperature(temperature, "top_logits")
    N, V = logits.shape
    k = int(k)
    if not 1 <= k <= min(V, _lib.TOP_LOGITS_MAX):
        raise ValueError(f"top_logits: k = {k} outside 1 .. {min(V, _lib.TOP_LOGITS_MAX)}")
    _gpu(logits, "top_logits")
    z = _dense(logits.detach())
    dev = z.device
    values = torch.empty(N, k, dtype=z.dtype, device=dev)
    ids = torch.empty(N, k, dtype=torch.int64, device=dev)
    rest = torch.empty(N, dtype=torch.float32, device=dev)
    if N:
        lib = _lib.load()
        with _on(dev):
            nb = lib.vln_top_logits_ws_bytes(N, V, _TYPES[z.dtype], k)
            ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
            _lib.check(lib.vln_top_logits(z.data_ptr(), _ld(z), _TYPES[z.dtype], N, V, k, T, values.data_ptr(), ids.data_ptr(), rest.data_ptr(),
                                          _p(ws), nb, _lib.raw_stream()), "vln_top_logits")
    return values, ids, rest


# ---- distillation ----------------------------------------------------------------------------------------------------------------
def _grad_like(z: torch.Tensor):
    """An uninitialised gradient for the rows `z`: where a row's distance from a 16-byte boundary changes from row to row (an odd
    vocabulary), the gradient's rows get the same distances, so that reads and writes can both take 16 bytes."""
    N, V = z.shape
    per = 16 // z.element_size()
    pad = (_ld(z) - V) % per
    return torch.empty(N, V + pad, dtype=z.dtype, device=z.device)[:, :V] if pad else torch.empty(N, V, dtype=z.dtype, device=z.device)


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, teacher, rest, target, T, alpha, ignore_index, reduction):
        z = _dense(logits.detach())
        N, V = z.shape
        dev = z.device
        lib = _lib.load()
        red = _lib.REDUCE[reduction]
        f32 = dict(dtype=torch.float32, device=dev)
        rows, stats = torch.empty(N, **f32), torch.empty(N, _lib.DISTILL_STATS, **f32)
        out = torch.empty(2, **f32) if red else None                # [loss, what the backward multiplies with]
        with _on(dev):
            a = _Distill.args(z, ids, teacher, rest, target, T, alpha, ignore_index, rows, stats)
            nb = lib.vln_distill_ws_bytes(N, V, a.type)
            ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
            _lib.check(lib.vln_distill_fwd(C.byref(a), red, _p(out), _p(ws), nb, _lib.raw_stream()), "vln_distill_fwd")
        ctx.save_for_backward(logits, ids, teacher, rest, target, rows, stats, out)
        ctx.cfg = (T, alpha, ignore_index, red)
        return out[0] if red else rows

    @staticmethod
    def args(z, ids, teacher, rest, target, T, alpha, ignore_index, rows, stats):
        return _lib.Distill(z.data_ptr(), _ld(z), ids.data_ptr(), _ld(ids), teacher.data_ptr(), _ld(teacher), _p(rest), _p(target),
                            ignore_index, rows.data_ptr(), stats.data_ptr(), T, alpha, _TYPES[z.dtype], _TYPES[teacher.dtype], z.shape[0],
                            z.shape[1], ids.shape[1], 0)

    @staticmethod
    def backward(ctx, dloss):
        logits, ids, teacher, rest, target, rows, stats, out = ctx.saved_tensors
        T, alpha, ignore_index, red = ctx.cfg
        z = _dense(logits.detach())
        dz = _grad_like(z)
        if red or dloss.stride(0) == 0:
            stride = 0
        else:
            stride, dloss = 1, dloss.contiguous()
        with _on(z.device):
            a = _Distill.args(z, ids, teacher, rest, target, T, alpha, ignore_index, rows, stats)
            _lib.check(_lib.load().vln_distill_bwd(C.byref(a), dloss.data_ptr(), stride, out.data_ptr() + 4 if red else None, dz.data_ptr(),
                                                   dz.stride(0), _lib.raw_stream()), "vln_distill_bwd")
        return dz, None, None, None, None, None, None, None, None


def distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_values: torch.Tensor, *, teacher_rest: Optional[torch.Tensor] = None,
                 temperature: float = 1.0, target: Optional[torch.Tensor] = None, alpha: float = 1.0, ignore_index: int = -1,
                 reduction: str = "mean") -> torch.Tensor:
    """A student's loss against the K words a teacher kept per row (`top_logits` of the teacher):

        alpha * T^2 * KL(teacher || student at temperature T)  +  (1 - alpha) * CrossEntropyLoss(logits, target)

    logits [N, V]; teacher_ids [N, K] int64 (outside [0, V): absent, e.g. -1), teacher_values [N, K] their logits (float32 / bfloat16),
    K <= 256.  teacher_rest [N] float32 = logsumexp(the teacher's other logits / T): then "any other word" is one more outcome, compared
    with the student's mass outside the kept words; None: the teacher is renormalised over the words it kept.  A word listed twice counts
    as two outcomes that share it.

    target [N] int64: needed for alpha < 1.  Rows whose target is `ignore_index` -- without targets, rows whose teacher has no mass --
    have loss and gradient 0 and do not count in the mean (no row counted: nan); a target outside [0, V) otherwise makes its row nan.
    With targets, a row whose teacher has no mass keeps its hard term.  A student that gives no mass to a word the teacher does has loss
    inf there.  reduction: "mean" over the counted rows, "sum" or "none" ([N]).

    One pass over the logits forward, one backward (logits in, gradient out); nothing of size [N, V] is kept in between.  Gradients go
    to `logits` only."""
    _rows(logits, "distill_loss")
    N, V = logits.shape
    dev = logits.device
    T = _temperature(temperature, "distill_loss")
    alpha = float(alpha)
    if not 0.0 <= alpha <= 1.0:
        raise ValueError(f"distill_loss: alpha {alpha} outside [0, 1]")
    if reduction not in _lib.REDUCE:
        raise ValueError("distill_loss: reduction must be 'none', 'sum' or 'mean'")
    if target is None and alpha < 1.0:
        raise ValueError("distill_loss: alpha < 1 needs targets")
    for t, name in ((teacher_values, "teacher_values"), (teacher_rest, "teacher_rest")):
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"distill_loss: {name} is a constant, it gets no gradient (detach it)")
    ids = _list(teacher_ids, N, dev, torch.int64, "distill_loss: teacher_ids")
    if teacher_values.dtype not in _TYPES:
        raise TypeError(f"distill_loss: teacher_values must be float32 or bfloat16, got {teacher_values.dtype}")
    tv = _list(teacher_values.detach(), N, dev, teacher_values.dtype, "distill_loss: teacher_values")
    if ids.shape != tv.shape or not 1 <= ids.shape[1] <= _lib.DISTILL_MAX:
        raise ValueError(f"distill_loss: teacher_ids {tuple(ids.shape)} and teacher_values {tuple(tv.shape)} must match, 1 .. {_lib.DISTILL_MAX} per row")
    ids, tv = _dense(ids), _dense(tv)
    rest = None if teacher_rest is None else _vector(teacher_rest, N, dev, torch.float32, "distill_loss: teacher_rest")
    tgt = None if target is None else _vector(target, N, dev, torch.int64, "distill_loss: target")
    _gpu(logits, "distill_loss")
    if N == 0:
        return logits.float().sum(1) if reduction == "none" else logits.float().sum() * (1.0 if reduction == "sum" else float("nan"))
    return _Distill.apply(logits, ids, tv, rest, tgt, T, alpha, int(ignore_index), reduction)
