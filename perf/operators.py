"""Measured cases of the word-head operators (vln_amd.vocab): constraints on word logits, a teacher's top logits, and the distillation
loss with its gradient -- each in a plain form of elementary torch operations and as the framework's own call."""
import math

import numpy as np
import torch

own = False          # True: run() makes the framework's calls; False: the plain forms below

_DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


# ---- cases -----------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # word-by-word decoding of ONE instruction with the speaker's 992-word vocabulary: pure latency
        dict(name="constrain_b1", op="constrain", N=1, V=992, dtype="fp32", H=20, P=0, bias=0, grammar=False, out=True, grad=False),
        # sampled training of the speaker (batch 64, 80 words so far): gradients run through the constrained logits
        dict(name="constrain_train_b64", op="constrain", N=64, V=992, dtype="fp32", H=80, P=0, bias=1, grammar=True, out=False, grad=True),
        # serving a batch of requests with prompts and word biases, an odd vocabulary
        dict(name="constrain_b256", op="constrain", N=256, V=32001, dtype="bf16", H=1024, P=512, bias=16, grammar=True, out=False, grad=False),
        # the largest decoding batch, long histories, into a fixed buffer
        dict(name="constrain_b512_large", op="constrain", N=512, V=131072, dtype="bf16", H=4096, P=0, bias=300, grammar=True, out=True, grad=False),
        # the greedy word of one decoding step
        dict(name="top_greedy_b64", op="top", N=64, V=992, dtype="fp32", K=1, T=1.0),
        # teacher targets of one speaker batch (64 instructions x 80 words)
        dict(name="top_speaker", op="top", N=5120, V=992, dtype="fp32", K=16, T=2.0),
        # candidates of a few beams over a large vocabulary: few rows, a long axis
        dict(name="top_beams", op="top", N=4, V=131072, dtype="fp32", K=128, T=1.0),
        # teacher targets over a large vocabulary
        dict(name="top_teacher_large", op="top", N=4096, V=32000, dtype="bf16", K=64, T=2.0),
        # the smallest training call: a short instruction, a few kept words
        dict(name="distill_small", op="distill", N=16, V=992, dtype="fp32", K=8, T=2.0, alpha=0.5, tail=False, empty=0.1),
        # one speaker batch, hard targets mixed in, the teacher's remaining mass as one more outcome
        dict(name="distill_speaker", op="distill", N=5120, V=992, dtype="fp32", K=16, T=2.0, alpha=0.7, tail=True, empty=0.2),
        # ragged: odd rows, an odd vocabulary
        dict(name="distill_odd", op="distill", N=1021, V=50001, dtype="bf16", K=33, T=1.0, alpha=1.0, tail=True, empty=0.05),
        # a long batch over a large vocabulary
        dict(name="distill_large", op="distill", N=8192, V=32000, dtype="bf16", K=64, T=2.0, alpha=0.5, tail=False, empty=0.05),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["constrain", "top", "distill"])
    V = _log_int(rng, 100, 131072)
    N = max(1, min(_log_int(rng, 1, 8192), (1 << 26) // V))
    dtype = rng.choice(["fp32", "bf16"])
    if op == "constrain":
        grad = rng.random() < 0.4
        return dict(op=op, N=min(N, 512), V=V, dtype=dtype, H=_log_int(rng, 1, 4096), P=rng.choice([0, _log_int(rng, 1, 2048)]),
                    bias=rng.choice([0, _log_int(rng, 1, 300)]), grammar=rng.random() < 0.6, out=not grad and rng.random() < 0.5, grad=grad)
    K = min(V // 2, _log_int(rng, 1, 128))
    T = rng.choice([1.0, 2.0, round(rng.uniform(0.5, 4.0), 2)])
    if op == "top":
        return dict(op=op, N=N, V=V, dtype=dtype, K=K, T=T)
    return dict(op=op, N=N, V=V, dtype=dtype, K=K, T=T, alpha=rng.choice([1.0, 0.5, round(rng.random(), 2)]), tail=rng.random() < 0.5,
                empty=rng.choice([0.0, 0.1, 0.3]))


def work(case):
    N, V, s = case["N"], case["V"], 4 if case["dtype"] == "fp32" else 2
    row = N * V * s
    if case["op"] == "constrain":
        lists = 8 * N * (case["H"] + case["P"]) + 12 * N * case["bias"] + (4 * N * ((V + 31) // 32) if case["grammar"] else 0)
        passes = 4 if case["grad"] else 2           # logits in, logits out; with gradients also the upstream in and the gradient out
        return {"bytes": passes * row + lists, "flops": N * V * (2 if case["grad"] else 1)}
    K = case["K"]
    if case["op"] == "top":
        return {"bytes": row + N * K * (s + 8) + 4 * N, "flops": 4 * N * V}
    return {"bytes": 2 * row + N * (K * 12 + 24), "flops": 10 * N * V}


# ---- inputs ----------------------------------------------------------------------------------------------------------------------
def _logits(g, N, V, dtype):
    """Word logits as a trained head gives them: a broad bulk and a few likely words per row."""
    dev = torch.device("cuda:0")
    z = torch.randn(N, V, generator=g, device=dev) * 1.5
    k = min(V, 24)
    start = torch.randint(0, V, (N, 1), generator=g, device=dev)
    hot = (start + (V // k) * torch.arange(k, device=dev)) % V          # distinct words
    z.scatter_(1, hot, torch.randn(N, k, generator=g, device=dev) * 2.0 + 6.0)
    return z.to(_DT[dtype])


def _ragged(g, N, n, V, dev):
    """[N, n] word ids, a few of them often, each row valid up to its own length (zero among them)."""
    ids = (torch.rand(N, n, generator=g, device=dev) ** 3 * V).long().clamp_(0, V - 1)
    lens = torch.randint(0, n + 1, (N,), generator=g, device=dev)
    lens[0] = n
    return ids, lens


def _inputs(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)
    N, V = case["N"], case["V"]
    x = {"logits": _logits(g, N, V, case["dtype"])}
    if case["op"] == "constrain":
        x["history"], x["history_lengths"] = _ragged(g, N, case["H"], V, dev)
        if case["P"]:
            x["prompt"], x["prompt_lengths"] = _ragged(g, N, case["P"], V, dev)
        x["repetition"] = 1.0 + torch.rand(N, generator=g, device=dev) * 0.5
        x["presence"] = torch.rand(N, generator=g, device=dev) * 0.6
        x["frequency"] = torch.rand(N, generator=g, device=dev) * 0.3
        if case["bias"]:
            x["bias_ids"] = torch.randint(0, V, (N, case["bias"]), generator=g, device=dev)
            x["bias_values"] = torch.randn(N, case["bias"], generator=g, device=dev) * 3.0
        if case["grammar"]:
            words = (V + 31) // 32
            G = min(N, 64)                   # states of the grammar; some allow almost nothing, some almost everything
            a = torch.randint(-2 ** 31, 2 ** 31, (G, words), generator=g, device=dev)
            b = torch.randint(-2 ** 31, 2 ** 31, (G, words), generator=g, device=dev)
            kind = torch.arange(G, device=dev).view(G, 1) % 4
            few = torch.where(torch.rand(G, words, generator=g, device=dev) < 0.02, a, torch.zeros_like(a))
            m = torch.where(kind == 0, few, torch.where(kind == 1, a & b, torch.where(kind == 2, a | b, torch.full_like(a, -1))))
            x["allowed"] = m.to(torch.int32)
            rows = torch.randint(0, G, (N,), generator=g, device=dev)
            rows[torch.rand(N, generator=g, device=dev) < 0.15] = -1          # requests without a grammar
            x["allowed_rows"] = rows
        if case["grad"]:
            x["upstream"] = (torch.randn(N, V, generator=g, device=dev) * 0.1).to(_DT[case["dtype"]])
        return x
    if case["op"] == "top":
        return x
    K, T = case["K"], case["T"]
    # the teacher saw the same text: its logits are the student's with other noise; it keeps K words and the mass of the others
    t = x["logits"].float() + torch.randn(N, V, generator=g, device=dev) * 0.7
    val, ids = torch.topk(t, K, dim=1)
    x["teacher_values"] = val.to(_DT[case["dtype"]])
    if case["tail"]:
        t.scatter_(1, ids, float("-inf"))
        x["teacher_rest"] = torch.logsumexp(t / T, 1)
    keep = torch.randint(1, K + 1, (N,), generator=g, device=dev)             # rows that kept fewer words: absent entries are -1
    short = torch.rand(N, generator=g, device=dev) < 0.25
    cut = short.view(N, 1) & (torch.arange(K, device=dev).view(1, K) >= keep.view(N, 1))
    x["teacher_ids"] = ids.masked_fill(cut, -1)
    target = ids[:, 0].clone()
    target[torch.rand(N, generator=g, device=dev) < case["empty"]] = -1       # padding of shorter texts
    target[0] = ids[0, 0]
    x["target"] = target
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    if case["op"] == "distill" or (case["op"] == "constrain" and case["grad"]):
        x["logits"].requires_grad_(True)
    if case["op"] == "constrain" and case["out"]:
        x["out"] = torch.empty_like(x["logits"])          # the fixed buffer that the decoder's next stage reads
    return {"case": case, "x": x}


# ---- plain forms -----------------------------------------------------------------------------------------------------------------
def _plain_constrain(case, x):
    z0 = x["logits"].detach()
    N, V = z0.shape
    z = z0.float()
    dev = z.device

    def counts(ids, lens):
        live = torch.arange(ids.shape[1], device=dev).view(1, -1) < lens.view(N, 1)
        return torch.zeros(N, V, device=dev).scatter_add_(1, ids, live.float())

    c = counts(x["history"], x["history_lengths"])
    seen = c > 0
    if "prompt" in x:
        seen = seen | (counts(x["prompt"], x["prompt_lengths"]) > 0)
    r = x["repetition"].view(N, 1)
    t = torch.where(seen, torch.where(z > 0, z / r, z * r), z)
    t = t - (x["frequency"].view(N, 1) * c + x["presence"].view(N, 1) * (c > 0))
    if "bias_ids" in x:
        t = t + torch.zeros(N, V, device=dev).scatter_add_(1, x["bias_ids"], x["bias_values"])
    ok = None
    if "allowed" in x:
        v = torch.arange(V, device=dev)
        rows = x["allowed_rows"]
        bits = x["allowed"][rows.clamp(min=0)][:, v >> 5]
        ok = (((bits >> (v & 31)) & 1) == 1) | (rows < 0).view(N, 1)
        t = torch.where(ok, t, torch.full_like(t, float("-inf")))
    out = t.to(z0.dtype)
    if not case["grad"]:
        return out
    up = x["upstream"].float()
    d = torch.where(seen, torch.where(z > 0, up / r, up * r), up)
    if ok is not None:
        d = torch.where(ok, d, torch.zeros_like(d))
    return out, d.to(z0.dtype)


def _plain_top(case, x):
    z = x["logits"]
    N, V = z.shape
    f = z.float()
    b = (f + 0.0).view(torch.int32)
    order = torch.where(b < 0, b ^ 0x7FFFFFFF, b).long()
    key = order * (1 << 32) + (V - 1 - torch.arange(V, device=z.device))      # larger value first, then the lower index
    ids = V - 1 - (torch.topk(key, case["K"], dim=1).values & 0xFFFFFFFF)
    values = z.gather(1, ids)
    u = f / case["T"]
    u.scatter_(1, ids, float("-inf"))
    m = u.max(1).values
    m0 = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    rest = m0 + (u - m0.view(N, 1)).exp().sum(1).log()
    return values, ids, rest


def _plain_distill(case, x):
    z0 = x["logits"].detach()
    N, V = z0.shape
    T, alpha = case["T"], case["alpha"]
    z = z0.float()
    u = z / T
    ids, present = x["teacher_ids"].clamp(min=0), x["teacher_ids"] >= 0
    ninf = float("-inf")
    t = torch.where(present, x["teacher_values"].float() / T, torch.full(ids.shape, ninf, device=z.device))
    if "teacher_rest" in x:
        t = torch.cat((t, x["teacher_rest"].view(N, 1)), 1)
    tm = t.max(1, keepdim=True).values
    logq = (t - tm) - (t - tm).exp().sum(1, keepdim=True).log()
    q = logq.exp()
    um = u.max(1, keepdim=True).values
    e = (u - um).exp()
    lse = um + e.sum(1, keepdim=True).log()
    zero = torch.zeros((), device=z.device)
    qw, lqw = q[:, :ids.shape[1]], logq[:, :ids.shape[1]]
    soft = torch.where(qw > 0, qw * (lqw - (u.gather(1, ids) - lse)), zero).sum(1)
    p = (u - lse).exp()
    grad = p - torch.zeros_like(p).scatter_add_(1, ids, qw)
    if "teacher_rest" in x:
        held = torch.zeros(N, V, device=z.device).scatter_add_(1, ids, present.float()) > 0
        w = torch.where(held, torch.full_like(u, ninf), u)
        wm = w.max(1, keepdim=True).values
        lrest = wm + (w - wm).exp().sum(1, keepdim=True).log()
        rr, lr = q[:, -1:], logq[:, -1:]
        soft = soft + torch.where(rr > 0, rr * (lr - (lrest - lse)), zero).view(N)
        grad = grad - rr * (w - lrest).exp()
    loss = alpha * T * T * soft
    grad = alpha * T * grad
    y = x["target"].clamp(min=0).view(N, 1)
    if alpha < 1.0:
        zm = z.max(1, keepdim=True).values
        l1 = zm + (z - zm).exp().sum(1, keepdim=True).log()
        loss = loss + (1 - alpha) * (l1 - z.gather(1, y)).view(N)
        hard = (z - l1).exp()
        hard.scatter_add_(1, y, torch.full((N, 1), -1.0, device=z.device))
        grad = grad + (1 - alpha) * hard
    live = x["target"] >= 0
    n = live.sum().float()
    loss = torch.where(live, loss, torch.zeros_like(loss)).sum() / n
    grad = torch.where(live.view(N, 1), grad / n, zero)
    return loss, grad.to(z0.dtype)


# ---- one pass --------------------------------------------------------------------------------------------------------------------
_PLAIN = {"constrain": _plain_constrain, "top": _plain_top, "distill": _plain_distill}
_LISTS = ("history", "history_lengths", "prompt", "prompt_lengths", "repetition", "presence", "frequency", "bias_ids", "bias_values", "allowed",
          "allowed_rows")


def run(state):
    case, x = state["case"], state["x"]
    if not own:
        return _PLAIN[case["op"]](case, x)
    from vln_amd import vocab
    if case["op"] == "top":
        return vocab.top_logits(x["logits"], case["K"], case["T"])
    if case["op"] == "distill":
        loss = vocab.distill_loss(x["logits"], x["teacher_ids"], x["teacher_values"], teacher_rest=x.get("teacher_rest"), temperature=case["T"],
                                  target=x["target"], alpha=case["alpha"])
        return loss.detach(), torch.autograd.grad(loss, x["logits"])[0]
    kw = {k: x[k] for k in _LISTS if k in x}
    if case["out"]:
        return vocab.constrain_logits(x["logits"], out=x["out"], **kw)
    out = vocab.constrain_logits(x["logits"], **kw)
    if not case["grad"]:
        return out
    return out.detach(), torch.autograd.grad(out, x["logits"], x["upstream"])[0]


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------------------------
def _exact_constrain(case, x):
    z = x["logits"].detach().double().cpu().numpy()
    N, V = z.shape
    h = {k: v.cpu().numpy() for k, v in x.items() if k != "logits" and k != "upstream"}
    up = x["upstream"].double().cpu().numpy() if case["grad"] else None
    out, dz = z.copy(), (up.copy() if up is not None else None)
    for b in range(N):
        hist, times = np.unique(h["history"][b, :h["history_lengths"][b]], return_counts=True)
        seen = hist
        if "prompt" in h:
            seen = np.union1d(hist, h["prompt"][b, :h["prompt_lengths"][b]])
        r = float(h["repetition"][b])
        zs = z[b, seen]
        out[b, seen] = np.where(zs > 0, zs / r, zs * r)
        if dz is not None:
            dz[b, seen] *= np.where(zs > 0, 1.0 / r, r)
        out[b, hist] -= float(h["frequency"][b]) * times + float(h["presence"][b])
        if "bias_ids" in h:
            np.add.at(out[b], h["bias_ids"][b], h["bias_values"][b].astype(np.float64))
        if "allowed" in h and h["allowed_rows"][b] >= 0:
            bits = np.unpackbits(h["allowed"][h["allowed_rows"][b]].view(np.uint8), bitorder="little")[:V]
            out[b, bits == 0] = -np.inf
            if dz is not None:
                dz[b, bits == 0] = 0.0
    o = torch.from_numpy(out)
    return o if dz is None else (o, torch.from_numpy(dz))


def _exact_top(case, x):
    z, K = x["logits"], case["K"]
    vals, idx, rest = [], [], []
    for part in z.split(max(1, (1 << 25) // z.shape[1])):
        v, i = torch.sort(part.double(), dim=1, descending=True, stable=True)
        vals.append(v[:, :K].cpu()); idx.append(i[:, :K].cpu())
        rest.append(torch.logsumexp(v[:, K:] / case["T"], 1).cpu() if K < z.shape[1] else torch.full((part.shape[0],), float("-inf"), dtype=torch.float64))
    return torch.cat(vals), torch.cat(idx), torch.cat(rest)


def _exact_distill(case, x):
    T, alpha = case["T"], case["alpha"]
    live = x["target"] >= 0
    n = int(live.sum())
    total, grads = 0.0, []
    step = max(1, (1 << 24) // case["V"])
    for a in range(0, case["N"], step):
        z = x["logits"].detach()[a:a + step].double()
        R, V = z.shape
        ids = x["teacher_ids"][a:a + step]
        logp = torch.log_softmax(z / T, 1)
        tq = (x["teacher_values"][a:a + step].double() / T).masked_fill(ids < 0, float("-inf"))
        if case["tail"]:
            tq = torch.cat((tq, x["teacher_rest"][a:a + step].double()[:, None]), 1)
        q = torch.softmax(tq, 1)
        # the teacher and the student as distributions over V words and one slot for "any other word"
        Q = torch.zeros(R, V + 1, dtype=torch.float64, device=z.device)
        Q.scatter_add_(1, ids.masked_fill(ids < 0, V), q[:, :ids.shape[1]])
        named = torch.zeros(R, V + 1, dtype=torch.bool, device=z.device).scatter_(1, ids.masked_fill(ids < 0, V), True)[:, :V]
        if case["tail"]:
            Q[:, V] = q[:, -1]
            other = logp.masked_fill(named, float("-inf"))
            LP = torch.cat((logp, torch.logsumexp(other, 1, keepdim=True)), 1)
            dz = torch.exp(logp) - Q[:, :V] - Q[:, V:] * torch.softmax(other, 1)
        else:
            LP = torch.cat((logp, torch.zeros(R, 1, dtype=torch.float64, device=z.device)), 1)
            dz = torch.exp(logp) - Q[:, :V]
        kl = torch.where(Q > 0, Q * (torch.log(Q.clamp_min(1e-300)) - LP), torch.zeros_like(Q)).sum(1)
        loss = alpha * T * T * kl
        dz = dz * (alpha * T)
        y = x["target"][a:a + step]
        hot = torch.zeros_like(z).scatter_(1, y.clamp(min=0)[:, None], 1.0)
        l1 = torch.log_softmax(z, 1)
        loss = loss - (1 - alpha) * (l1 * hot).sum(1)
        dz = dz + (1 - alpha) * (torch.exp(l1) - hot)
        keep = y >= 0
        total += float(loss[keep].sum())
        grads.append((dz * (keep.double() / n)[:, None]).cpu())
    return torch.tensor(total / n, dtype=torch.float64), torch.cat(grads)


def exact(case, seed):
    if case["N"] * case["V"] > 1 << 27 or (case["op"] == "constrain" and case["N"] * case["V"] > 1 << 25):
        return None          # too many numbers for the host in the time there is
    return {"constrain": _exact_constrain, "top": _exact_top, "distill": _exact_distill}[case["op"]](case, _inputs(case, seed))
