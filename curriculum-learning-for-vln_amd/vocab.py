"""Word logits [N, V] (the speaker's vocabulary head): what shapes them before a word is drawn, and what a student learns from a teacher's.

    constrain_logits   penalties for repeated words, word biases, grammar masks          (differentiable; in place for decoding)
    top_logits         the k largest logits of every row and the log-mass of the others  (a teacher's targets; k = 1: the greedy word)
    distill_loss       the loss of a student against such targets, with its gradient     (differentiable)

fp32 or bf16 logits, rows any distance apart; arithmetic in fp32, one rounding to the logits' type at the end.  There is no CPU
fallback.  Everything is launched on the current stream of the logits' device; nothing synchronises, nothing is kept between calls."""
from __future__ import annotations

import ctypes as C
import functools
from dataclasses import dataclass
from typing import Callable, Optional, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib, losses, ops

_TYPES = {torch.float32: ops.F32, torch.bfloat16: ops.BF16}
_byref = C.byref


def _launch(fn, name: str, device, *args):
    """fn(*args, stream) on the current stream of the logits' device, also when another device is current."""
    if device.index == _lib._get_device():
        st = fn(*args, _lib.raw_stream())
    else:
        with torch.cuda.device(device):
            st = fn(*args, _lib.raw_stream())
    if st:
        _lib.check(st, name)


def _rows(t: torch.Tensor, name: str):
    """(N, V, type code) of word logits [N, V]."""
    losses._not_deferred(t, name)
    code = _TYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name}: expected float32 or bfloat16 logits, got {t.dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name}: expected logits [N, V], got {tuple(t.shape)}")
    N, V = t.shape
    if V < 1 or N >= 1 << 31 or V >= 1 << 31:
        raise ValueError(f"{name}: expected logits [N, V] with 1 <= V < 2^31, got {tuple(t.shape)}")
    return N, V, code


def _gpu(t: torch.Tensor, name: str):
    if not t.is_cuda:
        raise _lib.VlnError(f"{name}: expected GPU tensors (the HIP path has no CPU fallback)")


def _dense(t: torch.Tensor, N: int, n: int):
    """`t` [N, n] if its rows are contiguous and do not overlap, else a copy that is such."""
    s0, s1 = t.stride()
    return t if (s1 == 1 or n == 1) and (s0 >= n or N == 1) else t.contiguous()


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
    if t.dim() != 1 or t.shape[0] != N:
        raise ValueError(f"{name}: expected [{N}], got {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _constant(t, name: str):
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} gets no gradient: it is a constant here (detach it)")


def _held(lists):
    """The lists a backward will read, with their versions: kept like this, not by save_for_backward, because a call's host time is mostly
    autograd's (and they are small; the logits, which are not, are saved and freed by autograd).  Tensors of inference mode have no version."""
    return [(t, None if t.is_inference() else t._version) for t in lists if t is not None]


def _unchanged(held):
    for t, version in held:
        if version is not None and t._version != version:
            raise RuntimeError(f"a tensor of shape {tuple(t.shape)} that the backward needs has been modified by an inplace operation "
                               f"(version {t._version}, expected {version})")


def _returned(ctx, N: int, V: int, code: int, device):
    """The forward's logits as autograd hands them back: a checkpoint or a saved-tensor hook returns another tensor, which has to be alike."""
    z, = ctx.saved_tensors
    if z.device != device or _TYPES.get(z.dtype) != code or z.dim() != 2 or z.shape[0] != N or z.shape[1] != V:
        raise RuntimeError(f"the saved logits came back as {tuple(z.shape)} {z.dtype} on {z.device}, they were [{N}, {V}] on {device}")
    return _dense(z, N, V)


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


def _constrain_call(src, dst, logits, args, device):
    """One launch over filled-in `args`; logits: the forward's input (the backward), or None."""
    setattr(args, "in", src.data_ptr())
    args.out = dst.data_ptr()
    args.ld_in, args.ld_out = max(src.stride(0), args.V), max(dst.stride(0), args.V)
    args.backward = 0
    if logits is not None:
        args.logits, args.ld_logits, args.backward = logits.data_ptr(), max(logits.stride(0), args.V), 1
    _launch(_lib.load().vln_constrain_logits, "vln_constrain_logits", device, _byref(args))


class _Constrain(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, args, lists):
        N, V = logits.shape
        z = _dense(logits, N, V)
        out = torch.empty(z.shape, dtype=z.dtype, device=z.device)
        _constrain_call(z, out, None, args, z.device)
        ctx.save_for_backward(logits)
        ctx.args, ctx.held = args, _held(lists)
        return out

    @staticmethod
    def backward(ctx, dout):
        return _Constrain.second(ctx, dout) if torch.is_grad_enabled() else _Constrain.first(ctx, dout)

    @staticmethod
    def first(ctx, dout):
        a = ctx.args
        z, d = _returned(ctx, a.B, a.V, a.type, dout.device), _dense(dout, a.B, a.V)
        _unchanged(ctx.held)
        dz = torch.empty(z.shape, dtype=z.dtype, device=z.device)
        _constrain_call(d, dz, z, a, z.device)
        return dz, None, None

    second = staticmethod(once_differentiable(first.__func__))       # (create_graph=True: a second derivative is an error)


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
    all); ids outside [0, V) -- padding: -1 -- stand for no word.  repetition (> 0, not subnormal) / presence / frequency: a number, or float32 [N].
    bias_ids int64 / bias_values float32: [N, n] or [n] for every row, n <= 2048; a word listed twice gets both.  allowed: int32 mask
    rows [G, ceil(V / 32)] from `pack_allowed`; allowed_rows int64 [N] picks each row's (-1: unconstrained; anything else outside [0, G)
    bans every word, which is visible, never a read out of range); without it G is N, or 1 for all.  A row whose mask allows nothing is
    -inf throughout.

    out: where to write (same shape and type; `logits` itself: in place, untouched words are not even read).  Without `out` the result
    carries gradients to `logits` (0 for banned words); penalties and biases are constants."""
    N, V, code = _rows(logits, "constrain_logits")
    dev = logits.device
    a, lists = _lib.Constrain(), []
    a.type, a.B, a.V = code, N, V
    if history is not None:
        _word_list(a, lists, history, history_lengths, N, dev, "history", "H")
    elif history_lengths is not None:
        raise ValueError("constrain_logits: history_lengths without history")
    if prompt is not None:
        _word_list(a, lists, prompt, prompt_lengths, N, dev, "prompt", "P")
    elif prompt_lengths is not None:
        raise ValueError("constrain_logits: prompt_lengths without prompt")
    for name, v in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if isinstance(v, torch.Tensor):
            _constant(v, "constrain_logits: " + name)
            v = _vector(v, N, dev, torch.float32, "constrain_logits: " + name)
            setattr(a, name, v.data_ptr())
            lists.append(v)
        else:
            v = float(v)
            if not abs(v) < float("inf") or name == "repetition" and v < 2.0 ** -126:
                raise ValueError(f"constrain_logits: {name} = {v}")
            setattr(a, name + "_all", v)
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("constrain_logits: bias_ids and bias_values belong together")
    if bias_ids is not None:
        _constant(bias_values, "constrain_logits: bias_values")
        bi = _list(bias_ids, N, dev, torch.int64, "constrain_logits: bias_ids", True)
        bv = _list(bias_values, N, dev, torch.float32, "constrain_logits: bias_values", True)
        n = bi.shape[1]
        if bv.shape[1] != n or n > _lib.CONSTRAIN_MAX_BIAS:
            raise ValueError(f"constrain_logits: bias_ids {tuple(bias_ids.shape)} and bias_values {tuple(bias_values.shape)} must match, "
                             f"at most {_lib.CONSTRAIN_MAX_BIAS} per row")
        if n:
            a.bias_ids, a.bias_values, a.n_bias, a.ld_bias_ids, a.ld_bias_values = bi.data_ptr(), bv.data_ptr(), n, bi.stride(0), bv.stride(0)
            lists += (bi, bv)
    if allowed is not None:
        words = (V + 31) // 32
        if allowed.dim() != 2 or allowed.shape[0] < 1 or allowed.shape[1] != words:
            raise ValueError(f"constrain_logits: allowed must be [G >= 1, {words}] for {V} words, got {tuple(allowed.shape)}")
        G = allowed.shape[0]
        al = _dense(_list(allowed, G, dev, torch.int32, "constrain_logits: allowed"), G, words)
        a.allowed, a.G, a.ld_allowed = al.data_ptr(), G, max(al.stride(0), words)
        lists.append(al)
        if allowed_rows is not None:
            rows = _vector(allowed_rows, N, dev, torch.int64, "constrain_logits: allowed_rows")
            a.allowed_rows = rows.data_ptr()
            lists.append(rows)
        elif G != 1 and G != N:
            raise ValueError(f"constrain_logits: {G} mask rows for {N} rows of logits need allowed_rows")
    elif allowed_rows is not None:
        raise ValueError("constrain_logits: allowed_rows without allowed")
    learns = logits.requires_grad and torch.is_grad_enabled()
    if out is None:
        _gpu(logits, "constrain_logits")
        if N == 0:
            return logits.clone()
        if learns:
            return _Constrain.apply(logits, a, lists)
        z = _dense(logits, N, V)
        out = torch.empty(z.shape, dtype=z.dtype, device=dev)
        _constrain_call(z, out, None, a, dev)
        return out
    if learns or out.requires_grad and torch.is_grad_enabled():
        raise ValueError("constrain_logits: out= carries no gradient; leave it out, or call under torch.no_grad()")
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev:
        raise ValueError(f"constrain_logits: out must be {tuple(logits.shape)} {logits.dtype} on {dev}")
    if N and (_dense(logits, N, V) is not logits or _dense(out, N, V) is not out):
        raise ValueError("constrain_logits: with out=, the rows of both tensors must be contiguous and must not overlap")
    ld_in, ld_out, p_in, p_out = max(logits.stride(0), V), max(out.stride(0), V), logits.data_ptr(), out.data_ptr()
    if N and not (p_in == p_out and (ld_in == ld_out or N == 1)):
        size = logits.element_size()
        if p_out < p_in + ((N - 1) * ld_in + V) * size and p_in < p_out + ((N - 1) * ld_out + V) * size:
            raise ValueError("constrain_logits: out overlaps the logits without being the same tensor")
    _gpu(logits, "constrain_logits")
    if N:
        _constrain_call(logits, out, None, a, dev)
        torch.autograd.graph.increment_version(out)          # (a graph that saved `out` must not use it as if it were unchanged)
    return out


def _word_list(a, lists, ids, lens, N, dev, name, size):
    """history / prompt: the struct's <name>, ld_<name>, <name>_len and the length H / P."""
    t = _list(ids, N, dev, torch.int64, "constrain_logits: " + name)
    n = t.shape[1]
    if n >= 1 << 31:
        raise ValueError(f"constrain_logits: {name} is longer than 2^31 words")
    if lens is not None:
        lens = _vector(lens, N, dev, torch.int64, f"constrain_logits: {name}_lengths")
    if n:
        setattr(a, name, t.data_ptr())
        setattr(a, "ld_" + name, t.stride(0))
        setattr(a, size, n)
        lists.append(t)
        if lens is not None:
            setattr(a, name + "_len", lens.data_ptr())
            lists.append(lens)


@dataclass
class WordConstraints:
    """The constraints of a whole decoding loop (`Speaker.infer_batch(constraints=...)`): constrain_logits' arguments, applied to every word
    with the words so far as the history.  allowed: mask rows (`pack_allowed`); next_rows(t, words [N, t] int64 on the device) -> int64 [N]
    on the device, each row's mask row for word t -- a grammar's state; None: mask row n (or the only one) throughout.  infer_batch adds one
    bias (<UNK>), so that at most 2047 are left."""
    repetition: Union[float, torch.Tensor] = 1.0
    presence: Union[float, torch.Tensor] = 0.0
    frequency: Union[float, torch.Tensor] = 0.0
    prompt: Optional[torch.Tensor] = None
    prompt_lengths: Optional[torch.Tensor] = None
    bias_ids: Optional[torch.Tensor] = None
    bias_values: Optional[torch.Tensor] = None
    allowed: Optional[torch.Tensor] = None
    next_rows: Optional[Callable[[int, torch.Tensor], torch.Tensor]] = None

    def banning(self, word: int, N: int, device) -> "WordConstraints":
        """The same constraints with one more word banned (a bias of -inf)."""
        ids = torch.full((N, 1), int(word), dtype=torch.int64, device=device)
        values = torch.full((N, 1), float("-inf"), device=device)
        if self.bias_ids is not None:
            ids = torch.cat((self.bias_ids.expand(N, -1), ids), 1)
            values = torch.cat((self.bias_values.expand(N, -1), values), 1)
        return WordConstraints(self.repetition, self.presence, self.frequency, self.prompt, self.prompt_lengths, ids, values, self.allowed, self.next_rows)

    def apply(self, logits: torch.Tensor, words: torch.Tensor) -> torch.Tensor:
        """constrain_logits for the word after `words` [N, t]."""
        rows = self.next_rows(words.shape[1], words) if self.next_rows is not None else None
        return constrain_logits(logits, history=words, prompt=self.prompt, prompt_lengths=self.prompt_lengths, repetition=self.repetition,
                                presence=self.presence, frequency=self.frequency, bias_ids=self.bias_ids, bias_values=self.bias_values,
                                allowed=self.allowed, allowed_rows=rows)


# ---- a teacher's top logits ------------------------------------------------------------------------------------------------------
def _temperature(T, who):
    T = float(T)
    if not _lib.TEMPERATURE_MIN <= T <= _lib.TEMPERATURE_MAX:
        raise ValueError(f"{who}: temperature {T} outside [{_lib.TEMPERATURE_MIN}, {_lib.TEMPERATURE_MAX}]")
    return T


@functools.lru_cache(maxsize=4096)
def _top_ws(device_index, N, V, code, k):          # (depends on the device's number of compute units)
    return _lib.load().vln_top_logits_ws_bytes(N, V, code, k)


@functools.lru_cache(maxsize=4096)
def _distill_ws(device_index, N, V, code):
    return _lib.load().vln_distill_ws_bytes(N, V, code)


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0):
    """(values [N, k], ids [N, k] int64, rest [N] float32): the k largest logits of every row, largest first, equal ones in the order of
    their ids (NaN counts as largest), and `rest = logsumexp(all other logits / temperature)` (-inf: none) -- the targets that
    `distill_loss` takes; `ids` with k = 1 is the greedy word.  1 <= k <= min(V, 256).  No gradient: a teacher is a constant."""
    N, V, code = _rows(logits, "top_logits")
    T = _temperature(temperature, "top_logits")
    k = int(k)
    if not 1 <= k <= min(V, _lib.TOP_LOGITS_MAX):
        raise ValueError(f"top_logits: k = {k} outside 1 .. {min(V, _lib.TOP_LOGITS_MAX)}")
    _gpu(logits, "top_logits")
    z = _dense(logits, N, V)
    dev = z.device
    values = torch.empty(N, k, dtype=z.dtype, device=dev)
    ids = torch.empty(N, k, dtype=torch.int64, device=dev)
    rest = torch.empty(N, dtype=torch.float32, device=dev)
    if N:
        nb = _top_ws(dev.index, N, V, code, k)
        ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        _launch(_lib.load().vln_top_logits, "vln_top_logits", dev, z.data_ptr(), max(z.stride(0), V), code, N, V, k, T, values.data_ptr(),
                ids.data_ptr(), rest.data_ptr(), ws.data_ptr() if nb else None, nb)
    return values, ids, rest


@dataclass
class DistillTargets:
    """What a teacher leaves for its student (`Speaker.teacher_targets`): top_logits' results for every row and the loss's settings."""
    ids: torch.Tensor
    values: torch.Tensor
    rest: Optional[torch.Tensor] = None
    temperature: float = 1.0
    alpha: float = 0.5


# ---- distillation ----------------------------------------------------------------------------------------------------------------
def _grad_like(z: torch.Tensor, N: int, V: int):
    """An uninitialised gradient for the rows `z`: where a row's distance from a 16-byte boundary changes from row to row (an odd
    vocabulary), the gradient's rows get the same distances, so that reads and writes can both take 16 bytes."""
    pad = (max(z.stride(0), V) - V) % (16 // z.element_size())
    return torch.empty(N, V + pad, dtype=z.dtype, device=z.device)[:, :V] if pad else torch.empty(N, V, dtype=z.dtype, device=z.device)


def _distill_forward(z, N, V, code, ids, teacher, rest, target, T, alpha, ignore_index, red):
    """(loss, the filled-in struct, the buffer it points to, 1 / count's address): all but the loss serve the backward as well."""
    dev = z.device
    # one buffer: the rows' statistics (16-byte aligned), 1 / count, and the rows' losses unless they are the result
    own_rows = N if red else 0
    buf = torch.empty(N * _lib.DISTILL_STATS + 4 + own_rows, dtype=torch.float32, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev) if red else torch.empty(N, dtype=torch.float32, device=dev)
    stats, out, K = buf.data_ptr(), loss.data_ptr(), ids.shape[1]
    inv = stats + 4 * N * _lib.DISTILL_STATS
    a = _lib.Distill(z.data_ptr(), max(z.stride(0), V), ids.data_ptr(), max(ids.stride(0), K), teacher.data_ptr(), max(teacher.stride(0), K),
                     None if rest is None else rest.data_ptr(), None if target is None else target.data_ptr(), ignore_index,
                     inv + 16 if red else out, stats, T, alpha, code, _TYPES[teacher.dtype], N, V, K, 0)
    nb = _distill_ws(dev.index, N, V, code)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
    _launch(_lib.load().vln_distill_fwd, "vln_distill_fwd", dev, _byref(a), red, out if red else None, inv if red else None,
            ws.data_ptr() if nb else None, nb)
    return loss, a, buf, inv if red else None


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, meta):
        z = _dense(logits, meta[0], meta[1])
        loss, ctx.args, ctx.buf, ctx.inv = _distill_forward(z, *meta)
        ctx.save_for_backward(z)
        ctx.held = _held(meta[3:7])
        return loss

    @staticmethod
    def backward(ctx, dloss):
        return _Distill.second(ctx, dloss) if torch.is_grad_enabled() else _Distill.first(ctx, dloss)

    @staticmethod
    def first(ctx, dloss):
        a, inv = ctx.args, ctx.inv
        z = _returned(ctx, a.N, a.V, a.type, dloss.device)
        a.logits, a.ld = z.data_ptr(), max(z.stride(0), a.V)
        _unchanged(ctx.held)
        dz = _grad_like(z, a.N, a.V)
        stride = 0
        if inv is None and dloss.stride(0) != 0:
            stride, dloss = 1, dloss.contiguous()
        _launch(_lib.load().vln_distill_bwd, "vln_distill_bwd", z.device, _byref(a), dloss.data_ptr(), stride, inv, dz.data_ptr(), dz.stride(0))
        return dz, None

    second = staticmethod(once_differentiable(first.__func__))       # (create_graph=True: a second derivative is an error)


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
    have loss and gradient 0 and do not count in the mean (no row counted: nan); with alpha < 1 any other target outside [0, V) makes its
    row nan.  With targets, a row whose teacher has no mass keeps its hard term.  A student that gives no mass to a word the teacher does has loss
    inf there.  reduction: "mean" over the counted rows, "sum" or "none" ([N]).

    One pass over the logits forward, one backward (logits in, gradient out); nothing of size [N, V] is kept in between.  Gradients go
    to `logits` only."""
    N, V, code = _rows(logits, "distill_loss")
    dev = logits.device
    T = _temperature(temperature, "distill_loss")
    alpha = float(alpha)
    if not 0.0 <= alpha <= 1.0:
        raise ValueError(f"distill_loss: alpha {alpha} outside [0, 1]")
    red = _lib.REDUCE.get(reduction)
    if red is None:
        raise ValueError("distill_loss: reduction must be 'none', 'sum' or 'mean'")
    if teacher_values.dtype not in _TYPES:
        raise TypeError(f"distill_loss: teacher_values must be float32 or bfloat16, got {teacher_values.dtype}")
    _constant(teacher_values, "distill_loss: teacher_values")
    ids = _list(teacher_ids, N, dev, torch.int64, "distill_loss: teacher_ids")
    tv = _list(teacher_values, N, dev, teacher_values.dtype, "distill_loss: teacher_values")
    K = ids.shape[1]
    if tv.shape[1] != K or not 1 <= K <= _lib.DISTILL_MAX:
        raise ValueError(f"distill_loss: teacher_ids {tuple(ids.shape)} and teacher_values {tuple(tv.shape)} must match, 1 .. {_lib.DISTILL_MAX} per row")
    ids, tv = _dense(ids, N, K), _dense(tv, N, K)
    if teacher_rest is not None:
        _constant(teacher_rest, "distill_loss: teacher_rest")
        teacher_rest = _vector(teacher_rest, N, dev, torch.float32, "distill_loss: teacher_rest")
    if target is not None:
        target = _vector(target, N, dev, torch.int64, "distill_loss: target")
    elif alpha < 1.0:
        raise ValueError("distill_loss: alpha < 1 needs targets")
    _gpu(logits, "distill_loss")
    if N == 0:
        return logits.float().sum(1) if reduction == "none" else logits.float().sum() * (1.0 if reduction == "sum" else float("nan"))
    meta = (N, V, code, ids, tv, teacher_rest, target, T, alpha, int(ignore_index), red)
    if logits.requires_grad and torch.is_grad_enabled():
        return _Distill.apply(logits, meta)
    return _distill_forward(_dense(logits, N, V), *meta)[0]
