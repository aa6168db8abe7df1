"""GPU: the word-logit operators (vln_amd.vocab) against plain 64-bit implementations of their definitions, at the sizes, strides and masks
where they can go wrong.

Tolerances are sums of half steps (`torch.finfo(t).eps / 2`, relative to the value: 2^-24 for fp32, 2^-8 for bf16), written beside each
comparison; U below is 2^-24."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
NINF = float("-inf")
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def vocab():
    import vln_amd
    vln_amd._lib.load()
    return vln_amd.vocab


def dev():
    return torch.device("cuda:0")


def place(t, how):
    """The CPU tensor on the GPU: plain, as a column slice of wider rows, or starting at an odd element."""
    if how == "plain":
        return t.to(dev())
    N, V = t.shape
    if how == "wide":
        w = torch.full((N, V + 13), float("nan"), dtype=t.dtype, device=dev())
        w[:, :V] = t.to(dev())
        return w[:, :V]
    flat = torch.full((N * V + 3,), float("nan"), dtype=t.dtype, device=dev())
    v = flat[3:].view(N, V)
    v.copy_(t)
    return v


def close(got, ref, tol, what):
    """|got - ref| <= tol elementwise; infinities and NaN where the reference has them."""
    got, ref, tol = got.detach().double().cpu(), ref.double(), torch.as_tensor(tol, dtype=torch.float64).expand(ref.shape)
    assert got.shape == ref.shape, f"{what}: {tuple(got.shape)} vs {tuple(ref.shape)}"
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in other places"
    inf = torch.isinf(ref)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], ref[inf]), f"{what}: infinities in other places"
    ok = ~inf & ~torch.isnan(ref)
    bad = (got - ref).abs()[ok] > tol[ok]
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got - ref).abs()[ok] / tol[ok].clamp_min(1e-300)).max():.2f} x the bound"


# ---- constraints ---------------------------------------------------------------------------------------------------------------------
def constrain64(z, hist=None, prompt=None, r=None, p=None, f=None, bias=None, ok=None, dout=None):
    """Row by row from the definition.  hist / prompt / bias: per row a list of ids (bias: of (id, value)).  Returns (out, scale, d z): scale =
    the sum of the absolute values of the terms that were added, for the tolerance."""
    N, V = z.shape
    out = z.double().clone()
    scale = out.abs()
    dz = None if dout is None else dout.double().clone()
    for b in range(N):
        h = [i for i in (hist[b] if hist else []) if 0 <= i < V]
        seen = set(h) | {i for i in (prompt[b] if prompt else []) if 0 <= i < V}
        count = {}
        for i in h:
            count[i] = count.get(i, 0) + 1
        for v in seen:
            x = float(z[b, v])
            t = x / r[b] if x > 0 else x * r[b]
            if dz is not None:
                dz[b, v] *= 1.0 / r[b] if x > 0 else r[b]
            c = count.get(v, 0)
            if c:
                t -= f[b] * c + p[b]
            out[b, v] = t
            scale[b, v] = abs(x / r[b] if x > 0 else x * r[b]) + (abs(f[b] * c) + abs(p[b]) if c else 0.0)
        for i, w in (bias[b] if bias else []):
            if 0 <= i < V:
                out[b, i] += w
                scale[b, i] += abs(w)
        if ok is not None:
            out[b, ~ok[b]] = NINF
            if dz is not None:
                dz[b, ~ok[b]] = 0.0
    return out, scale, dz


def constrain_case(N, V, H, P, nb, grammar, seed):
    g = torch.Generator().manual_seed(seed)
    # ids from -3 to V + 2: a few stand for no word, and small vocabularies repeat them often
    ids = lambda n: torch.randint(-3, V + 3, (N, n), generator=g)
    lens = lambda n: torch.randint(0, n + 1, (N,), generator=g)
    c = dict(history=ids(H), history_lengths=lens(H), prompt=ids(P), prompt_lengths=lens(P),
             repetition=1.0 + torch.rand(N, generator=g), presence=torch.rand(N, generator=g), frequency=torch.rand(N, generator=g) * 0.5)
    if nb:
        c["bias_ids"], c["bias_values"] = ids(nb), torch.randn(N, nb, generator=g) * 4
    ok = None
    if grammar:
        ok = torch.rand(N + 2, V, generator=g) < 0.6
        ok[0] = False                                  # a state that allows nothing
        rows = torch.randint(-1, N + 2, (N,), generator=g)
        rows[0] = 0
        if N > 2:
            rows[1], rows[2] = N + 2, -2               # outside the mask rows: no word is allowed
        c["mask"], c["allowed_rows"] = ok, rows
        full = torch.ones(N, V, dtype=torch.bool)
        for b in range(N):
            q = int(rows[b])
            full[b] = ok[q] if 0 <= q < N + 2 else q == -1
        ok = full
    hist = [c["history"][b, :int(c["history_lengths"][b])].tolist() for b in range(N)]
    prom = [c["prompt"][b, :int(c["prompt_lengths"][b])].tolist() for b in range(N)]
    bias = [list(zip(c["bias_ids"][b].tolist(), c["bias_values"][b].double().tolist())) for b in range(N)] if nb else None
    ref = dict(hist=hist, prompt=prom, r=c["repetition"].double().tolist(), p=c["presence"].double().tolist(), f=c["frequency"].double().tolist(),
               bias=bias, ok=ok)
    return c, ref


def call_args(vocab, c):
    kw = {k: v.to(dev()) for k, v in c.items() if k != "mask"}
    if "mask" in c:
        kw["allowed"] = vocab.pack_allowed(c["mask"].to(dev()))
    return kw


def constrain_tol(dt, ref, scale, nb):
    # quotient or product, f * c, + p, the difference: 4 roundings of at most the terms' sum; nb additions of biases; 1 rounding to bf16
    t = (4 + nb) * U * scale
    return t + (0 if dt == torch.float32 else 2.0 ** -8 * (ref.abs().nan_to_num(0, 0, 0) + t)) + 1e-40


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("how", ["plain", "wide", "odd"])
@pytest.mark.parametrize("N,V,H,P,nb,grammar", [(1, 1, 1, 1, 1, False), (3, 7, 5, 0, 3, True), (4, 31, 40, 9, 20, True), (5, 64, 0, 0, 0, True),
                                                (2, 992, 80, 30, 0, False), (6, 1003, 300, 40, 200, True), (3, 20011, 700, 100, 50, True),
                                                (2, 40000, 9000, 5000, 2048, False)])
def test_constrain_logits(vocab, N, V, H, P, nb, grammar, how, dt):
    c, ref = constrain_case(N, V, H, P, nb, grammar, 7 * N + V + H)
    g = torch.Generator().manual_seed(V)
    z = (torch.randn(N, V, generator=g) * 3).to(DT[dt])
    z[0, 0] = 0.0
    up = torch.randn(N, V, generator=g).to(DT[dt])
    out_ref, scale, dz_ref = constrain64(z, dout=up, **ref)
    zd = place(z, how)
    leaf = zd.detach().requires_grad_(True)
    kw = call_args(vocab, c)
    out = vocab.constrain_logits(leaf, **kw)
    tol = constrain_tol(DT[dt], out_ref, scale, nb)
    close(out, out_ref, tol, "out")
    dz, = torch.autograd.grad(out, leaf, place(up, how))
    # one quotient or product, and the rounding to bf16
    close(dz, dz_ref, (U + (0 if dt == "fp32" else 2.0 ** -8)) * 1.01 * dz_ref.abs() + 1e-40, "d logits")
    # into another tensor and in place: the same bits, and nothing outside the rows is touched
    buf = torch.full((N, V + 5), 7.0, dtype=DT[dt], device=dev())
    got = vocab.constrain_logits(zd, out=buf[:, 2:V + 2], **kw)
    assert torch.equal(got, out) and got.data_ptr() == buf[:, 2:].data_ptr()
    assert (buf[:, :2] == 7).all() and (buf[:, V + 2:] == 7).all()
    vocab.constrain_logits(zd, out=zd, **kw)
    assert torch.equal(zd, out)


def test_constrain_gradient_against_differences(vocab):
    """The map is linear around a point away from 0: (f(z + h e) - f(z - h e)) / 2h of the 64-bit definition is the gradient; the kernel's is
    one rounding off the formula, the differences are exact to 1e-9."""
    N, V = 2, 23
    c, ref = constrain_case(N, V, 12, 4, 5, False, 3)
    z = torch.randn(N, V, generator=torch.Generator().manual_seed(0))
    z = torch.where(z.abs() < 0.05, torch.full_like(z, 0.5), z)
    up = torch.randn(N, V, generator=torch.Generator().manual_seed(1))
    leaf = z.to(dev()).requires_grad_(True)
    dz, = torch.autograd.grad(vocab.constrain_logits(leaf, **call_args(vocab, c)), leaf, up.to(dev()))
    h = 1e-4
    num = torch.zeros(N, V, dtype=torch.float64)
    for b in range(N):
        for v in range(V):
            e = torch.zeros(N, V, dtype=torch.float64)
            e[b, v] = h
            hi, lo = constrain64(z.double() + e, **ref)[0], constrain64(z.double() - e, **ref)[0]
            num[b, v] = ((hi - lo) * up.double()).sum() / (2 * h)
    close(dz, num, 2 * U * num.abs() + 1e-9, "d logits")


@pytest.mark.parametrize("H", [16383, 16384, 32767, 32768, 70000])
def test_constrain_long_histories(vocab, H):
    """One word all the time: counts on both sides of the 14- and 15-bit counters, and past 16 bits."""
    V = 40
    z = torch.ones(2, V, device=dev())
    hist = torch.full((2, H), 5, dtype=torch.int64, device=dev())
    hist[1, ::2] = 39
    out = vocab.constrain_logits(z, history=hist, prompt=torch.tensor([[5], [-1]], device=dev()), frequency=0.25, presence=1.0, repetition=2.0)
    ref = torch.ones(2, V, dtype=torch.float64)
    ref[0, 5] = 0.5 - (0.25 * H + 1)
    ref[1, 39], ref[1, 5] = 0.5 - (0.25 * ((H + 1) // 2) + 1), 0.5 - (0.25 * (H // 2) + 1)
    close(out, ref, 4 * U * ref.abs() + 4 * U, "out")


def test_constrain_special_values(vocab):
    """NaN and infinities stay what the arithmetic makes of them where a word is allowed, and become -inf where it is banned; a banned word's
    gradient is 0 whatever the upstream holds."""
    lowest = torch.finfo(torch.float32).min
    z = torch.tensor([[float("nan"), float("inf"), NINF, lowest, 0.0, -0.0, 1.0, -1.0]]).repeat(2, 1)
    hist = torch.arange(8).repeat(2, 1)
    mask = torch.ones(2, 8, dtype=torch.bool)
    mask[1] = False
    leaf = z.to(dev()).requires_grad_(True)
    out = vocab.constrain_logits(leaf, history=hist.to(dev()), repetition=2.0, allowed=vocab.pack_allowed(mask.to(dev())))
    ref = torch.tensor([float("nan"), float("inf"), NINF, NINF, 0.0, 0.0, 0.5, -2.0]).double()      # lowest * 2 leaves the range
    close(out[0], ref, 0.0, "allowed")
    assert (out[1] == NINF).all()
    dz, = torch.autograd.grad(out, leaf, torch.full_like(out, float("nan")))
    assert torch.isnan(dz[0]).all() and (dz[1] == 0).all()
    up = torch.ones_like(out)
    dz, = torch.autograd.grad(vocab.constrain_logits(leaf, history=hist.to(dev()), repetition=2.0), leaf, up)
    assert dz[0, 1:].tolist() == [0.5, 2.0, 2.0, 2.0, 2.0, 0.5, 2.0]


def test_constrain_shared_lists_and_scalars(vocab):
    """[n] biases and one mask row for every row, a slice of a longer word buffer as the history (rows far apart), numbers for tensors."""
    N, V, T = 5, 992, 17
    g = torch.Generator().manual_seed(0)
    z = torch.randn(N, V, generator=g)
    words = torch.randint(0, V, (N, 120), generator=g)
    ok = torch.rand(1, V, generator=g) < 0.5
    bi, bv = torch.tensor([3, 3, 500, 991]), torch.tensor([1.0, 2.0, -4.0, 0.5])
    ref, scale, _ = constrain64(z, hist=[words[b, :T].tolist() for b in range(N)], r=[1.25] * N, p=[0.5] * N, f=[0.125] * N,
                                bias=[list(zip(bi.tolist(), bv.tolist()))] * N, ok=ok.expand(N, V))
    out = vocab.constrain_logits(z.to(dev()), history=words.to(dev())[:, :T], repetition=1.25, presence=0.5, frequency=0.125, bias_ids=bi.to(dev()),
                                 bias_values=bv.to(dev()), allowed=vocab.pack_allowed(ok).to(dev()))
    close(out, ref, constrain_tol(torch.float32, ref, scale, 4), "out")
    assert torch.equal(vocab.constrain_logits(z.to(dev())), z.to(dev()))              # no constraint: the logits
    assert vocab.constrain_logits(z.to(dev())[:0]).shape == (0, V)


# ---- a teacher's top logits ------------------------------------------------------------------------------------------------------------
def rank64(z):
    """Order of a row's elements: NaN first, then larger values, equal ones by index."""
    key = z.double().clone()
    nan = torch.isnan(key)
    return sorted(range(z.numel()), key=lambda i: (not bool(nan[i]), -float(key[i]) if not bool(nan[i]) else 0.0, i))


def check_top(vocab, z, k, T, how="plain"):
    N, V = z.shape
    values, ids, rest = vocab.top_logits(place(z, how), k, T)
    assert values.dtype == z.dtype and ids.dtype == torch.int64 and rest.dtype == torch.float32
    values, ids, rest = values.cpu(), ids.cpu(), rest.cpu()
    zd = z.double()
    if not torch.isnan(zd).any():
        sv, si = torch.sort(zd, dim=1, descending=True, stable=True)      # (+0 and -0 are equal, so is their order by index)
        want, other = si[:, :k], sv[:, k:]
    else:
        order = torch.tensor([rank64(z[b]) for b in range(N)])
        want, other = order[:, :k], zd.gather(1, order[:, k:])
    assert torch.equal(ids, want), [(b, ids[b].tolist()[:8], want[b].tolist()[:8]) for b in range(N) if not torch.equal(ids[b], want[b])][:3]
    got = values.double()
    exp = zd.gather(1, want)
    assert torch.equal(torch.isnan(got), torch.isnan(exp)) and torch.equal(got.nan_to_num(0, 1e39, -1e39), exp.nan_to_num(0, 1e39, -1e39))
    if k < V:
        ref = torch.logsumexp(other / T, 1)
        m = (other.max(1).values / T).nan_to_num(0, 0, 0).abs()
        # m / T and its sum with the logarithm: 4 half steps of each; in the exponents 4 half steps of (m - x) / T, whose mean under the
        # softmax is at most log V; v_exp (2), 16 terms per partial sum, one partial sum and at most one rescaling (3) per 1024 elements,
        # the lanes' tree and the segments' merge (32)
        tol = U * (4 * m + 4 * ref.abs().nan_to_num(0, 0, 0) + 4 * math.log(V) + 50 + 4 * V / 1024)
        close(rest, ref, tol, "rest")
    else:
        assert (rest == NINF).all()


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("N,V,k", [(1, 1, 1), (3, 5, 5), (2, 63, 7), (4, 64, 64), (3, 65, 64), (5, 992, 1), (5, 992, 16), (3, 1003, 65), (2, 1025, 128),
                                   (2, 5000, 129), (3, 9001, 256), (2, 300, 256), (1, 131072, 128), (2, 100003, 40), (17, 32001, 64)])
def test_top_logits(vocab, N, V, k, dt):
    g = torch.Generator().manual_seed(N * 1000 + V + k)
    z = (torch.randn(N, V, generator=g) * 2).to(DT[dt])               # bf16: many equal values
    check_top(vocab, z, k, 1.0)
    check_top(vocab, z, k, 2.5, "odd")
    check_top(vocab, z, k, 0.5, "wide")


@pytest.mark.parametrize("V,k", [(70, 16), (992, 16), (3000, 64), (20000, 256), (40001, 100)])
def test_top_logits_orders_and_ties(vocab, V, k):
    """Ascending rows (every chunk beats all before it), descending ones, constant rows, two values, masked rows with fewer than k words
    left, rows of -inf only, zeros of both signs."""
    up = torch.arange(V, dtype=torch.float32)
    two = (torch.arange(V) % 3 == 0).float()
    few = torch.full((V,), NINF)
    few[V // 2:V // 2 + 5] = torch.tensor([1.0, 3.0, 3.0, 2.0, 1.0])
    low = torch.full((V,), torch.finfo(torch.float32).min)
    low[3] = 1.0
    signs = torch.zeros(V)
    signs[::2] = -0.0
    z = torch.stack((up, -up, torch.zeros(V), torch.full((V,), -7.5), two, few, torch.full((V,), NINF), low, signs, -signs * up))
    check_top(vocab, z, k, 1.0)
    check_top(vocab, z.to(torch.bfloat16), k, 2.0)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("N,V,k", [(3, 992, 16), (4, 5003, 256), (2, 70001, 64), (600, 2500, 40), (2, 70001, 1)])
def test_top_logits_of_masked_rows(vocab, N, V, k, dt):
    """Rows in which a grammar left fewer words than are asked for, or a few in one place, or none: equal values (-inf, 0) fill the rest in
    index order, across vectors, waves and segments."""
    g = torch.Generator().manual_seed(V + k)
    z = torch.randn(N, V, generator=g).to(DT[dt])
    for b in range(N):
        left = [0, 1, k // 2, 2 * k, V // 50][b % 5]
        keep = torch.randperm(V, generator=g)[:left] if b % 2 else torch.arange(V // 3, min(V, V // 3 + left))
        m = torch.full((V,), NINF, dtype=z.dtype)
        m[keep] = z[b, keep]
        z[b] = m
    z[-1] = torch.where(torch.isinf(z[-1]), torch.zeros_like(z[-1]), z[-1].abs())      # ties at a finite value
    check_top(vocab, z, k, 1.0)
    check_top(vocab, z, k, 2.0, "odd")
    quantised = (torch.randn(N, V, generator=g) * 2).round().to(DT[dt])                # a dozen different values
    check_top(vocab, quantised, k, 1.0, "odd")


def test_top_logits_nan_and_infinities(vocab):
    V = 3000
    g = torch.Generator().manual_seed(4)
    z = torch.randn(6, V, generator=g)
    z[0, 77] = float("nan")
    z[1, ::50] = float("nan")                      # more NaN than k
    z[2, 5] = float("inf")
    z[3, 100:104] = float("inf")
    z[4] = float("nan")
    z[5, 2999], z[5, 0] = float("nan"), -float("nan")
    values, ids, rest = (t.cpu() for t in vocab.top_logits(z.to(dev()), 8, 1.0))
    for b in range(6):
        want = rank64(z[b])[:8]
        assert ids[b].tolist() == want, b
    assert torch.isnan(values[4]).all() and torch.isnan(rest[1]) and torch.isnan(rest[4])
    assert not torch.isnan(rest[[0, 2, 3, 5]]).any()
    close(rest[:1], torch.logsumexp(torch.cat((z[0, :77], z[0, 78:])).double().sort(descending=True).values[7:], 0).view(1), 200 * U, "rest beside a NaN")


def test_top_logits_many_rows(vocab):
    """More rows than the chip has waves: one wave per row; and no gradient is asked for."""
    g = torch.Generator().manual_seed(9)
    z = torch.randn(5120, 992, generator=g)
    check_top(vocab, z, 16, 2.0)
    assert not vocab.top_logits(z.to(dev()).requires_grad_(True), 3)[0].requires_grad
    v, i, r = vocab.top_logits(z.to(dev())[:0], 3)
    assert v.shape == (0, 3) and i.shape == (0, 3) and r.shape == (0,)


# ---- distillation --------------------------------------------------------------------------------------------------------------------
def distill64(z, ids, tv, rest, T, target, alpha, ignore=-1):
    """Row losses, counted rows, d rows / d z in 64 bits, and bounds for what fp32 may add (tol_row, tol_grad)."""
    N, V = z.shape
    z = z.double()
    loss, live = torch.zeros(N, dtype=torch.float64), torch.zeros(N, dtype=torch.bool)
    grad, tl, tg = torch.zeros_like(z), torch.zeros(N, dtype=torch.float64), torch.zeros_like(z)
    steps = 64 + 8 * V / 1024                       # roundings of a sum over a row (16 terms, partial sums, rescalings, tree) and of logarithms
    for b in range(N):
        y = None if target is None else int(target[b])
        out = [(int(i), float(t) / T) for i, t in zip(ids[b], tv[b].double()) if 0 <= int(i) < V]
        R = float(rest[b]) if rest is not None else NINF
        # relative to the largest before any logarithm is added: next to 3e38 even 64 bits lose it
        top = max([u for _, u in out] + [R])
        soft = top > NINF
        if soft:
            out, R = [(i, u - top) for i, u in out], R - top
        mass = [u for _, u in out] + [R]
        live[b] = soft if target is None else y != ignore
        if not live[b]:
            continue
        zt = (z[b] - (z[b].max() if z[b].max() > NINF else 0.0)) / T
        lse = float(torch.logsumexp(zt, 0))
        p = torch.exp(zt - lse)
        dist = (z[b].max() - z[b]).clamp(max=1e4).nan_to_num(1e4, 1e4, 1e4)
        rho = U * (steps + 8 * dist / T)            # relative error of p_v: its exponent carries 4 half steps of the distance, twice
        if soft and alpha > 0:
            L = float(torch.logsumexp(torch.tensor(mass, dtype=torch.float64), 0))
            kept = torch.zeros(V, dtype=torch.bool)
            qv = torch.zeros(V, dtype=torch.float64)
            for i, u in out:
                kept[i] = True
                q = math.exp(u - L)
                qv[i] += q
                if q > 0:
                    lp = float(zt[i]) - lse
                    loss[b] += alpha * T * T * q * ((u - L) - lp)
                    if lp > NINF:
                        tl[b] += alpha * T * T * q * float(U * (2 * steps + 8 * dist[i] / T + 8 * abs(u - max(mass)))) * (1 + abs(u - L - lp))
            r = math.exp(R - L)
            g = p - qv
            tgs = p * rho + qv * U * (steps + 8 * max(0.0, max(mass) - min([m for m in mass if m > NINF], default=0.0)))
            if r > 0:
                other = torch.where(kept, torch.full_like(zt, NINF), zt)
                lr = float(torch.logsumexp(other, 0))
                loss[b] += alpha * T * T * r * ((R - L) - (lr - lse))
                if lr > NINF:
                    tl[b] += alpha * T * T * r * U * (3 * steps + 8 * abs(R - max(mass)) + 8 * abs(lr - lse)) * (1 + abs(R - L - lr + lse))
                    share = torch.exp(other - lr)
                    g = g - r * share
                    tgs = tgs + r * share * (rho + U * (steps + 8 * abs(R - max(mass))))
            grad[b] += alpha * T * g
            tg[b] += alpha * T * tgs
        if alpha < 1:
            if not 0 <= y < V:
                loss[b], grad[b] = float("nan"), float("nan")
                continue
            z1 = zt * T
            l1 = float(torch.logsumexp(z1, 0))
            p1 = torch.exp(z1 - l1)
            loss[b] += (1 - alpha) * (l1 - float(z1[y]))
            tl[b] += (1 - alpha) * U * (steps + 4 * abs(l1 - float(z1[y])) + 4 * float(dist[y]))
            p1y = p1.clone()
            p1y[y] -= 1
            grad[b] += (1 - alpha) * p1y
            tg[b] += (1 - alpha) * (p1 * U * (steps + 8 * dist))
            tg[b, y] += (1 - alpha) * 4 * U
    return loss, live, grad, tl, tg


def check_distill(vocab, z, ids, tv, rest=None, T=1.0, target=None, alpha=1.0, how="plain", ignore=-1):
    loss, live, grad, tl, tg = distill64(z, ids, tv, rest, T, target, alpha, ignore)
    n = int(live.sum())
    on = lambda t: None if t is None else t.to(dev())
    leaf = place(z, how).detach().requires_grad_(True)
    kw = dict(teacher_rest=on(rest), temperature=T, target=on(target), alpha=alpha, ignore_index=ignore)
    half = 0.0 if z.dtype == torch.float32 else 2.0 ** -8

    rows = vocab.distill_loss(leaf, on(ids), on(tv), reduction="none", **kw)
    close(rows, loss, 1.01 * tl + 8 * U * loss.abs().nan_to_num(0, 0, 0) + 1e-30, "rows")
    w = torch.randn(z.shape[0], generator=torch.Generator().manual_seed(1))
    dz, = torch.autograd.grad(rows, leaf, on(w))
    bound = lambda s, ref: 1.02 * s.abs() * tg + (8 * U + half) * ref.abs().nan_to_num(0, 0, 0) + 1e-37
    close(dz, grad * w.double()[:, None], bound(w.double()[:, None], grad * w.double()[:, None]), "d logits (rows)")
    if n:
        mean = vocab.distill_loss(leaf, on(ids), on(tv), **kw)
        ok = torch.isfinite(loss)
        if ok.all():
            close(mean.view(1), (loss.sum() / n).view(1), 1.01 * tl.sum() / n + U * (z.shape[0] / 1024 + 30) * loss.abs().sum() / n + 1e-30, "mean")
        dz, = torch.autograd.grad(mean, leaf)
        close(dz, grad / n, bound(torch.tensor(1.0 / n), grad / n), "d logits (mean)")
        total = vocab.distill_loss(leaf, on(ids), on(tv), reduction="sum", **kw)
        if ok.all():
            close(total.view(1), loss.sum().view(1), 1.01 * tl.sum() + U * (z.shape[0] / 1024 + 30) * loss.abs().sum() + 1e-30, "sum")
    return rows, dz


def distill_case(N, V, K, dt, seed, tail, absent=0.2):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(N, V, generator=g) * 2).to(DT[dt])
    t = z.float() + torch.randn(N, V, generator=g)
    tv, ids = torch.topk(t, K, dim=1)
    rest = None
    if tail:
        rest = torch.logsumexp(t.scatter(1, ids, NINF), 1)
    ids = ids.masked_fill(torch.rand(N, K, generator=g) < absent, -1)
    target = torch.randint(0, V, (N,), generator=g)
    target[1::3] = -1
    if N > 2:
        target[2] = max(int(ids[2, 0]), 0)
    return z, ids, tv.to(DT[dt]), rest, target


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("T,alpha", [(1.0, 1.0), (2.0, 0.5), (1.0, 0.3), (0.5, 0.0), (3.0, 1.0)])
@pytest.mark.parametrize("N,V,K,how", [(1, 2, 1, "plain"), (5, 9, 4, "odd"), (4, 65, 64, "wide"), (7, 992, 16, "plain"), (6, 1003, 100, "odd"),
                                       (3, 20011, 256, "plain"), (2, 70000, 33, "wide")])
def test_distill_loss(vocab, N, V, K, how, T, alpha, tail, dt):
    z, ids, tv, rest, target = distill_case(N, V, K, dt, N + V + K, tail)
    check_distill(vocab, z, ids, tv, rest, T, target if alpha < 1 or V > 60 else None, alpha, how)


@pytest.mark.parametrize("tail", [False, True])
def test_distill_many_rows_and_no_targets(vocab, tail):
    """One wave per row; the mean counts the rows whose teacher has mass."""
    z, ids, tv, rest, _ = distill_case(5000, 130, 8, "fp32", 5, tail)
    ids[::7] = -1
    if tail:
        rest[::14] = NINF
    check_distill(vocab, z, ids, tv, rest, 2.0)


def test_distill_words_listed_twice(vocab):
    """Two outcomes that share a word: their probabilities add up in the gradient, the word counts once in the student's mass."""
    z, ids, tv, rest, target = distill_case(6, 300, 12, "fp32", 8, True, absent=0.0)
    ids[:, 5] = ids[:, 2]
    ids[3, :] = ids[3, 0]
    check_distill(vocab, z, ids, tv, rest, 2.0, target, 0.4)
    check_distill(vocab, z, ids, tv, None, 1.0)


def test_distill_empty_and_masked_rows(vocab):
    """Teachers without mass, masked students, the lowest finite value in masked places, ids outside the vocabulary, targets outside it."""
    V, K = 100, 6
    lowest = torch.finfo(torch.float32).min
    g = torch.Generator().manual_seed(2)
    z = torch.randn(9, V, generator=g)
    tv, ids = torch.topk(z + torch.randn(9, V, generator=g), K, dim=1)
    rest = torch.full((9,), -1.0)
    ids[0] = -1                       # row 0: nothing kept, nothing else: no mass
    rest[0] = NINF
    tv[1] = NINF                      # row 1: kept words without mass, the others have it
    z[2, ids[2]] = NINF               # row 2: the student bans what the teacher wants: loss inf
    z[3, ids[3][3:]] = NINF           # row 3: bans words to which the teacher gives no mass either
    tv[3, 3:] = NINF
    tv[4] = lowest                    # row 4: everything masked with the lowest value: equal shares
    rest[4] = NINF
    z[5] = lowest                     # row 5: a student that is masked throughout is uniform
    ids[6, 0], ids[6, 1] = V, 2 ** 40  # row 6: not words
    z[7] = NINF                       # row 7: a student without any mass
    z[7, 50] = 0.0
    target = torch.randint(0, V, (9,), generator=g)
    target[8] = -1
    z[8] = float("nan")               # row 8: ignored, whatever it holds
    for T in (1.0, 0.5):
        check_distill(vocab, z, ids, tv, rest, T, target, 1.0)
        check_distill(vocab, z[:7], ids[:7], tv[:7], None, T)
    # hard terms beside teachers without mass; a target outside the vocabulary is visible, an ignored row is not
    target[1] = V + 3
    rows, _ = check_distill(vocab, z[:2], ids[:2], tv[:2], rest[:2], 2.0, target[:2], 0.5)
    assert torch.isfinite(rows[0]) and torch.isnan(rows[1])
    rows, dz = check_distill(vocab, z[8:], ids[8:], tv[8:], rest[8:], 2.0, target[8:], 0.5)
    assert rows.tolist() == [0.0] and (dz == 0).all()
    all_ignored = torch.full((3,), -1)
    leaf = z[:3].to(dev()).requires_grad_(True)
    mean = vocab.distill_loss(leaf, ids[:3].to(dev()), tv[:3].to(dev()), target=all_ignored.to(dev()))
    assert torch.isnan(mean) and (torch.autograd.grad(mean, leaf)[0] == 0).all()
    # a NaN in the teacher makes its row NaN
    tv[4, 0] = float("nan")
    assert torch.isnan(vocab.distill_loss(z[4:5].to(dev()), ids[4:5].to(dev()), tv[4:5].to(dev())))
    # no rows
    for red, want in (("sum", 0.0), ("mean", float("nan"))):
        got = vocab.distill_loss(leaf[:0], ids[:0].to(dev()), tv[:0].to(dev()), reduction=red)
        assert got.dim() == 0 and (got == want or torch.isnan(got) == math.isnan(want))


def test_distill_student_without_any_mass(vocab):
    """A row of -inf only: no word has probability, so the loss against a teacher with mass is inf and the gradient is -q."""
    V = 70
    z = torch.full((1, V), NINF)
    ids, tv = torch.tensor([[3, 9]]), torch.tensor([[0.0, 0.0]])
    for rest in (None, torch.tensor([0.0])):
        leaf = z.to(dev()).requires_grad_(True)
        loss = vocab.distill_loss(leaf, ids.to(dev()), tv.to(dev()), teacher_rest=None if rest is None else rest.to(dev()), reduction="sum")
        assert loss == float("inf")
        dz, = torch.autograd.grad(loss, leaf)
        q = 0.5 if rest is None else 1.0 / 3.0
        ref = torch.zeros(1, V, dtype=torch.float64)
        ref[0, 3] = ref[0, 9] = -q
        close(dz, ref, 8 * U, "d logits")


def test_distill_sure_student_keeps_the_others_mass(vocab):
    """The student's mass outside the kept words is e^-60 of the whole: 1 - (kept mass) would be 0; here it is a sum of its own."""
    V = 500
    z = torch.randn(1, V, generator=torch.Generator().manual_seed(0)) - 60.0
    z[0, 7] = 5.0
    check_distill(vocab, z, torch.tensor([[7]]), torch.tensor([[1.0]]), torch.tensor([0.5]), 1.0)
    check_distill(vocab, z * 3, torch.tensor([[7]]), torch.tensor([[1.0]]), torch.tensor([0.5]), 1.0, torch.tensor([7]), 0.5)


def test_distill_gradient_against_differences(vocab):
    """Central differences of the 64-bit loss, step 1e-5: exact to about 1e-9 for losses of this size."""
    N, V, K = 3, 21, 5
    z, ids, tv, rest, target = distill_case(N, V, K, "fp32", 11, True)
    target[1] = 4
    leaf = z.to(dev()).requires_grad_(True)
    loss = vocab.distill_loss(leaf, ids.to(dev()), tv.to(dev()), teacher_rest=rest.to(dev()), temperature=2.0, target=target.to(dev()), alpha=0.6)
    dz, = torch.autograd.grad(loss, leaf)
    f = lambda x: distill64(x, ids, tv, rest, 2.0, target, 0.6)[0].mean()
    num = torch.zeros(N, V, dtype=torch.float64)
    for b in range(N):
        for v in range(V):
            e = torch.zeros(N, V, dtype=torch.float64)
            e[b, v] = 1e-5
            num[b, v] = (f(z.double() + e) - f(z.double() - e)) / 2e-5
    close(dz, num, 200 * U + 1e-8, "d logits")


# ---- how they are used -----------------------------------------------------------------------------------------------------------------
def pipeline(vocab, student, teacher, words, packed):
    """Decode a word under constraints, take the teacher's targets under the same ones, distil."""
    kw = dict(history=words, repetition=1.3, presence=0.2, frequency=0.1, allowed=packed)
    tv, ids, rest = vocab.top_logits(vocab.constrain_logits(teacher, **kw), 12, 2.0)
    tgt = ids[:, 0]
    out = vocab.constrain_logits(student, **kw)
    loss = vocab.distill_loss(out, ids, tv, teacher_rest=rest, temperature=2.0, target=tgt, alpha=0.7)
    dz, = torch.autograd.grad(loss, student)
    return loss.detach(), dz, ids


def pipeline_inputs(seed, N=6, V=5003):
    g = torch.Generator().manual_seed(seed)
    s, t = torch.randn(N, V, generator=g).to(dev()), torch.randn(N, V, generator=g).to(dev())
    return s.requires_grad_(True), t, torch.randint(0, V, (N, 30), generator=g).to(dev()), torch.rand(N, V, generator=g) < 0.9


def test_pipeline_against_the_definitions(vocab):
    s, t, words, mask = pipeline_inputs(0)
    loss, dz, ids = pipeline(vocab, s, t, words, vocab.pack_allowed(mask).to(dev()))
    N = s.shape[0]
    args = dict(hist=words.tolist(), r=[1.3] * N, p=[0.2] * N, f=[0.1] * N, ok=mask)
    s64, t64 = constrain64(s.detach().cpu(), **args)[0], constrain64(t.cpu(), **args)[0]
    order = torch.sort(t64, dim=1, descending=True, stable=True)
    assert torch.equal(ids.cpu(), order.indices[:, :12])
    rest = torch.logsumexp(order.values[:, 12:] / 2.0, 1)
    rows, _, grad, tl, tg = distill64(s64, order.indices[:, :12], order.values[:, :12], rest, 2.0, order.indices[:, 0], 0.7)
    # the constrained logits come with 4 half steps of their own (|z| < 8): 32 U more in every exponent
    close(loss.view(1), rows.mean().view(1), tl.mean() + 400 * U * (1 + rows.mean()), "loss")
    gz = constrain64(s.detach().cpu(), dout=grad / N, **args)[2]
    close(dz, gz, 1.3 * tg / N + 100 * U * gz.abs() + 1e-12, "d logits")


def test_graphs_and_streams(vocab):
    """Two captured graphs of the whole chain, replayed several times with eager work in between and on two streams at once, against eager
    results: bit for bit (no float atomics anywhere, and no scratch memory that two calls share)."""
    sets = [pipeline_inputs(i) for i in (1, 2)]
    packed = [vocab.pack_allowed(m).to(dev()) for *_, m in sets]
    graphs = []
    side = torch.cuda.Stream()
    for (s, t, w, _), pk in zip(sets, packed):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            pipeline(vocab, s, t, w, pk)
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = pipeline(vocab, s, t, w, pk)
        graphs.append((gr, res))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(4):
        new = [pipeline_inputs(10 + 2 * rep + i) for i in (0, 1)]
        with torch.no_grad():
            for (s, t, w, _), (s2, t2, w2, _) in zip(sets, new):
                s.copy_(s2); t.copy_(t2); w.copy_(w2)
        want = [tuple(x.clone() for x in pipeline(vocab, s, t, w, pk)) for (s, t, w, _), pk in zip(sets, packed)]
        torch.cuda.synchronize()
        for (gr, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for (_, got), ref in zip(graphs, want):
            for a, b in zip(got, ref):
                assert torch.equal(a, b)


def test_same_inputs_same_bits(vocab):
    z, ids, tv, rest, target = distill_case(700, 5001, 40, "bf16", 3, True)
    ids[:, 7] = ids[:, 3]
    c, _ = constrain_case(64, 5001, 200, 20, 100, True, 1)
    kw = call_args(vocab, c)
    leaf = z.to(dev()).requires_grad_(True)
    first = None
    for _ in range(3):
        loss = vocab.distill_loss(leaf, ids.to(dev()), tv.to(dev()), teacher_rest=rest.to(dev()), temperature=2.0, target=target.to(dev()), alpha=0.5)
        now = (loss.detach(), torch.autograd.grad(loss, leaf)[0], *vocab.top_logits(leaf, 40), vocab.constrain_logits(leaf[:64], **kw).detach())
        if first is None:
            first = now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


def test_upstream_gradients_and_repeated_backward(vocab):
    """Another upstream than 1, an expanded one, a second backward through the same forward."""
    z, ids, tv, rest, target = distill_case(9, 500, 10, "fp32", 6, False)
    leaf = z.to(dev()).requires_grad_(True)
    args = (ids.to(dev()), tv.to(dev()))
    loss = vocab.distill_loss(leaf, *args, reduction="sum")
    one, = torch.autograd.grad(loss, leaf, retain_graph=True)
    two, = torch.autograd.grad(loss, leaf, torch.tensor(2.0, device=dev()))
    assert torch.equal(two, 2 * one)
    rows = vocab.distill_loss(leaf, *args, reduction="none")
    assert torch.equal(torch.autograd.grad(rows.sum(), leaf)[0], one)


def test_calls_that_autograd_must_refuse(vocab):
    """A list or a target changed in place between forward and backward, logits overwritten through out= while a graph holds them, and a second
    derivative: errors, not wrong numbers."""
    z, ids, tv, rest, target = distill_case(5, 300, 6, "fp32", 4, True)
    leaf = z.to(dev()).requires_grad_(True)
    ids, tv = ids.to(dev()), tv.to(dev())
    loss = vocab.distill_loss(leaf, ids, tv)
    ids.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, leaf)
    hist = torch.zeros(5, 4, dtype=torch.int64, device=dev())
    out = vocab.constrain_logits(leaf, history=hist, repetition=2.0)
    hist[0, 0] = 3
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.sum(), leaf)
    w = (leaf * 1.0)
    y = (w * w).sum()                              # the product's backward needs w
    with torch.no_grad():
        vocab.constrain_logits(w, history=hist, repetition=2.0, out=w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaf)
    loss = vocab.distill_loss(leaf, ids, tv)
    g, = torch.autograd.grad(loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), leaf)


def test_rows_far_apart(vocab):
    """Rows whose offsets pass 2^31 elements (and 2^32 bytes): views of one large buffer."""
    V, ld = 1003, (1 << 30) + 7
    buf = torch.empty(2 * ld + V, dtype=torch.bfloat16, device=dev())
    z = buf.as_strided((3, V), (ld, 1))
    g = torch.Generator().manual_seed(0)
    zc = torch.randn(3, V, generator=g).to(torch.bfloat16)
    z.copy_(zc)
    hist = torch.randint(0, V, (3, 20), generator=g)
    packed = zc.to(dev())
    kw = dict(history=hist.to(dev()), repetition=1.5, frequency=0.5)
    assert torch.equal(vocab.constrain_logits(z, **kw), vocab.constrain_logits(packed, **kw))
    for a, b in zip(vocab.top_logits(z, 9, 2.0), vocab.top_logits(packed, 9, 2.0)):
        assert torch.equal(a, b)
    val, ids = torch.topk(zc.float(), 5, dim=1)
    res = []
    for x in (z, packed):
        leaf = x.detach().requires_grad_(True)
        loss = vocab.distill_loss(leaf, ids.to(dev()), val.to(dev()))
        res.append((loss.detach(), torch.autograd.grad(loss, leaf)[0]))
    assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])
    want = vocab.constrain_logits(packed, **kw)
    vocab.constrain_logits(z, out=z, **kw)
    assert torch.equal(z, want)


def test_on_another_stream(vocab):
    """Inputs made on one stream, the calls on another that waits for it."""
    z, ids, tv, rest, target = distill_case(64, 5001, 16, "bf16", 9, True)
    side = torch.cuda.Stream()
    leaf = z.to(dev()).requires_grad_(True)
    args = (ids.to(dev()), tv.to(dev()))
    want = vocab.distill_loss(leaf, *args, teacher_rest=rest.to(dev()), temperature=2.0)
    wg, = torch.autograd.grad(want, leaf)
    top = vocab.top_logits(leaf, 5)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = vocab.distill_loss(leaf, *args, teacher_rest=rest.to(dev()), temperature=2.0)
        gg, = torch.autograd.grad(got, leaf)
        top2 = vocab.top_logits(leaf, 5)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(want, got) and torch.equal(wg, gg) and all(torch.equal(a, b) for a, b in zip(top, top2))


def test_saved_logits_that_come_back_elsewhere(vocab):
    """Checkpoints (the chain is run again in the backward) and logits that wait on the CPU: the backward reads the tensor that autograd hands
    back, not the forward's address.  Teachers from inference mode have no version to compare."""
    from torch.utils.checkpoint import checkpoint
    z, ids, tv, rest, target = distill_case(33, 5001, 6, "bf16", 5, True)
    leaf = z.to(dev()).requires_grad_(True)
    hist = ids.to(dev())
    with torch.inference_mode():
        ids, tv, rest = ids.to(dev()) + 0, tv.to(dev()) * 1, rest.to(dev()) * 1

    def chain(x):
        y = vocab.constrain_logits(x * 1.0, history=hist, repetition=1.5, frequency=0.1)
        return vocab.distill_loss(y * 1.0, ids, tv, teacher_rest=rest, temperature=2.0)

    want, = torch.autograd.grad(chain(leaf), leaf)
    assert bool(want.ne(0).any())
    loss = checkpoint(chain, leaf, use_reentrant=False)
    trash = [torch.full((33, 5001), float("nan"), dtype=torch.bfloat16, device=dev()) for _ in range(8)]
    assert torch.equal(torch.autograd.grad(loss, leaf)[0], want)
    with torch.autograd.graph.save_on_cpu():
        loss = chain(leaf)
    trash += [torch.full((33, 5001), float("nan"), dtype=torch.bfloat16, device=dev()) for _ in range(8)]
    assert torch.equal(torch.autograd.grad(loss, leaf)[0], want)


def test_repetition_divides_like_a_division(vocab):
    """fp32, one repeated word in every row, penalties and logits over the whole range: the quotient's bits are a division's wherever it is a
    normal number; an overflow and infinite logits stay infinite."""
    g = torch.Generator().manual_seed(3)
    N = 4000
    r = torch.exp2(torch.rand(N, generator=g) * 240 - 120)
    z = torch.exp2(torch.rand(N, 1, generator=g) * 240 - 120)
    r[:1000], z[:1000] = torch.rand(1000, generator=g) + 1.0, torch.rand(1000, 1, generator=g) * 20       # the usual ones
    r[1000:1004] = torch.tensor([2.0 ** -126, 3.4e38, 1.0, 0.5])
    z[1000:1004, 0], z[1004, 0] = 3.4e38, float("inf")
    want = z[:, 0] / r
    got = vocab.constrain_logits(z.to(dev()), history=torch.zeros(N, 1, dtype=torch.int64, device=dev()), repetition=r.to(dev()))[:, 0].cpu()
    ok = (want >= 2.0 ** -126) | torch.isinf(want)
    assert int(ok.sum()) > 3000 and torch.equal(got[ok], want[ok])
    assert bool((got[~ok] <= 2.0 ** -126).all())


def test_saved_logits_that_come_back_different(vocab):
    """A hook that returns the saved logits in another type or shape: an error before any launch."""
    leaf = torch.randn(6, 500, device=dev()).requires_grad_(True)
    hist, ids, tv = torch.zeros(6, 3, dtype=torch.int64, device=dev()), torch.zeros(6, 1, dtype=torch.int64, device=dev()), torch.zeros(6, 1, device=dev())
    for back in (lambda t: t.bfloat16(), lambda t: t[:, :100], lambda t: t[0], lambda t: t.cpu()):
        for call in (lambda: vocab.constrain_logits(leaf, history=hist, repetition=2.0).sum(), lambda: vocab.distill_loss(leaf, ids, tv)):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: back(t) if t.dim() == 2 and t.shape == leaf.shape else t):
                loss = call()
            with pytest.raises(RuntimeError, match="came back"):
                torch.autograd.grad(loss, leaf)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("V,k", [(1100, 1), (2100, 16), (4001, 64), (4001, 65), (7000, 16), (7000, 128), (16001, 32), (31001, 64), (31001, 256), (65001, 40)])
def test_top_logits_of_unlike_units(vocab, V, k, dt):
    """Row lengths between the forms (registers of one wave, units of one, two and four waves, whole and cut), and rows in which a few units
    of eight hold what decides: one word far above all others, runs of large words, infinities and NaN beside ordinary words, words left
    by a mask of -inf or of the type's lowest value, rows that fall and rise."""
    t = DT[dt]
    g = torch.Generator().manual_seed(V + k)
    z = torch.randn(12, V, generator=g)
    z[1, V // 3] = 200.0
    z[2, V // 2:V // 2 + 2 * k] += 30.0
    z[3, 8 * (torch.randperm(V // 8, generator=g)[:min(k, 3)])] = float("inf")
    z[4, torch.randperm(V, generator=g)[:min(k, 3)]] = float("nan")
    z[5, torch.rand(V, generator=g) < 0.98] = NINF
    z[6, torch.rand(V, generator=g) < 0.98] = torch.finfo(t).min
    z[7] = torch.linspace(-30, 30, V)
    z[8] = torch.linspace(30, -30, V)
    z[9, 5:] = -90.0 + z[9, 5:]
    z[10] = torch.where(torch.arange(V) % 8 == 3, z[10].abs() + 5, z[10] - 50)       # the largest of every unit in one place
    z[11, :V - 3] = NINF
    z = z.to(t)
    others = z[torch.arange(12) != 4]
    for T, how in ((1.0, "plain"), (0.05, "odd"), (40.0, "wide")):
        check_top(vocab, others, k, T, how)
        check_top(vocab, z[4:5], k, T, how)
