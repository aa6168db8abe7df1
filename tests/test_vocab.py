"""CPU: what the word-logit operators (vln_amd.vocab) refuse, at the Python entry points and at the C ABI (argument checks come before any
device call), and the packing of grammar masks."""
import ctypes as C
import os

import pytest
import torch


@pytest.fixture(scope="module")
def vln():
    import vln_amd
    if not os.path.exists(vln_amd.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    return vln_amd


def test_pack_allowed():
    from vln_amd import vocab
    g = torch.Generator().manual_seed(0)
    for V in (1, 31, 32, 33, 992, 1003):
        mask = torch.rand(3, V, generator=g) < 0.5
        mask[0] = True
        packed = vocab.pack_allowed(mask)
        assert packed.dtype == torch.int32 and packed.shape == (3, (V + 31) // 32)
        v = torch.arange(V)
        assert torch.equal(((packed[:, v // 32].long() >> (v % 32)) & 1).bool(), mask)
    with pytest.raises(TypeError):
        vocab.pack_allowed(torch.ones(2, 3))


def test_cpu_tensors_are_refused(vln):
    z = torch.randn(2, 8)
    ids, val = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    for call in (lambda: vln.vocab.constrain_logits(z), lambda: vln.vocab.constrain_logits(z, out=z), lambda: vln.vocab.top_logits(z, 2),
                 lambda: vln.vocab.distill_loss(z, ids, val)):
        with pytest.raises(vln.VlnError, match="no CPU fallback"):
            call()


def test_constrain_refusals(vln):
    f = vln.vocab.constrain_logits
    z = torch.randn(2, 40)
    i64 = lambda *s: torch.zeros(*s, dtype=torch.int64)
    packed = torch.zeros(2, 2, dtype=torch.int32)
    bad_type, bad_value = [], []
    bad_type += [lambda: f(z.half()), lambda: f(z.double()), lambda: f(z, history=i64(2, 3).int()), lambda: f(z, bias_ids=i64(2, 1), bias_values=torch.zeros(2, 1).double()),
                 lambda: f(z, allowed=packed.long()), lambda: f(z, repetition=torch.ones(2).double()), lambda: f(z, history=i64(2, 3), history_lengths=i64(2).int())]
    bad_value += [lambda: f(z[0]), lambda: f(torch.zeros(2, 0)), lambda: f(z, history=i64(3, 3)), lambda: f(z, history=i64(3)), lambda: f(z, history_lengths=i64(2)),
                  lambda: f(z, prompt=i64(2, 3), prompt_lengths=i64(3)), lambda: f(z, repetition=0.0), lambda: f(z, repetition=-1.0),
                  lambda: f(z, repetition=float("nan")), lambda: f(z, presence=float("inf")), lambda: f(z, repetition=torch.ones(3)),
                  lambda: f(z, presence=torch.ones(2, requires_grad=True)), lambda: f(z, bias_ids=i64(2, 1)), lambda: f(z, bias_ids=i64(2, 1), bias_values=torch.zeros(2, 2)),
                  lambda: f(z, bias_ids=i64(2, 2049), bias_values=torch.zeros(2, 2049)), lambda: f(z, bias_ids=i64(1), bias_values=torch.zeros(1, requires_grad=True)),
                  lambda: f(z, allowed=packed[:, :1]), lambda: f(z, allowed_rows=i64(2)), lambda: f(z, allowed=torch.zeros(3, 2, dtype=torch.int32)),
                  lambda: f(z, allowed=packed, allowed_rows=i64(3)), lambda: f(z, out=torch.zeros(2, 41)), lambda: f(z, out=z.bfloat16()),
                  lambda: f(z.clone().requires_grad_(True), out=torch.zeros(2, 40)), lambda: f(z, out=torch.zeros(40, 2).t())]
    flat = torch.zeros(200)
    bad_value += [lambda: f(flat[:80].view(2, 40), out=flat[10:90].view(2, 40)), lambda: f(z[:1].expand(2, 40), out=torch.zeros(2, 40)),
                  lambda: f(flat[:80].view(2, 40), out=flat.as_strided((2, 40), (50, 1)))]
    for call in bad_type:
        with pytest.raises(TypeError):
            call()
    for call in bad_value:
        with pytest.raises(ValueError):
            call()


def test_top_logits_refusals(vln):
    f = vln.vocab.top_logits
    z = torch.randn(2, 400)
    for k in (0, -1, 257, 401):
        with pytest.raises(ValueError):
            f(z, k)
    with pytest.raises(ValueError):
        f(z[:, :5], 6)
    for T in (0.0, -1.0, float("nan"), float("inf"), 1e-4):
        with pytest.raises(ValueError):
            f(z, 3, T)
    with pytest.raises(TypeError):
        f(z.half(), 3)
    with pytest.raises(ValueError):
        f(z.view(1, 2, 400), 3)


def test_distill_refusals(vln):
    f = vln.vocab.distill_loss
    z, ids, tv = torch.randn(2, 40), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    tgt = torch.zeros(2, dtype=torch.int64)
    for call in (lambda: f(z, ids, tv, temperature=0.0), lambda: f(z, ids, tv, alpha=0.5), lambda: f(z, ids, tv, alpha=1.5, target=tgt),
                 lambda: f(z, ids, tv, alpha=float("nan"), target=tgt), lambda: f(z, ids, tv, reduction="max"), lambda: f(z, ids[:, :2], tv),
                 lambda: f(z, ids[:1], tv[:1]), lambda: f(z, ids[:, :0], tv[:, :0]), lambda: f(z, torch.zeros(2, 257, dtype=torch.int64), torch.zeros(2, 257)),
                 lambda: f(z, ids, tv, teacher_rest=torch.zeros(3)), lambda: f(z, ids, tv, target=tgt[:1]), lambda: f(z, ids, tv.clone().requires_grad_(True)),
                 lambda: f(z, ids, tv, teacher_rest=torch.zeros(2, requires_grad=True)), lambda: f(z.view(-1), ids, tv)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: f(z.half(), ids, tv), lambda: f(z, ids.int(), tv), lambda: f(z, ids, tv.half()), lambda: f(z, ids, tv, teacher_rest=torch.zeros(2).double()),
                 lambda: f(z, ids, tv, target=tgt.int())):
        with pytest.raises(TypeError):
            call()


def test_c_abi_refusals(vln):
    """Wrong sizes, missing pointers and unknown types end in VLN_ERR_ARG with a text, before any launch (the pointers here are not device
    memory and are never read)."""
    lib, L = vln._lib.load(), vln._lib
    p = 4096

    def constrain(**kw):
        a = L.Constrain()
        setattr(a, "in", p)
        a.out, a.ld_in, a.ld_out, a.B, a.V = p, 40, 40, 2, 40
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.vln_constrain_logits(C.byref(a), None)

    for kw in (dict(B=0), dict(V=0), dict(H=-1), dict(H=3), dict(P=2), dict(out=None), dict(ld_in=39), dict(ld_out=39), dict(backward=1), dict(n_bias=1),
               dict(n_bias=2049, bias_ids=p, bias_values=p), dict(allowed=p, G=0, ld_allowed=2), dict(allowed=p, G=2, ld_allowed=1),
               dict(allowed=p, G=3, ld_allowed=2), dict(type=7)):
        assert constrain(**kw) == 1, kw
        assert b"vln_constrain_logits" in lib.vln_last_error_string()
    assert lib.vln_constrain_logits(None, None) == 1

    def top(logits=p, ld=40, type=0, N=2, V=40, k=3, T=1.0, values=p, ids=p, rest=p, ws=None, nb=0):
        return lib.vln_top_logits(logits, ld, type, N, V, k, T, values, ids, rest, ws, nb, None)

    for kw in (dict(logits=None), dict(ld=39), dict(type=2), dict(N=0), dict(V=0), dict(k=0), dict(k=41), dict(T=0.0), dict(T=float("nan")), dict(rest=None),
               dict(V=131072, ld=131072, k=5)):                # the last: segments need a workspace
        assert top(**kw) == 1, kw
        assert b"vln_top_logits" in lib.vln_last_error_string()
    assert top(V=1000, ld=1000, k=257) == 1
    assert lib.vln_top_logits_ws_bytes(1, 131072, 0, 128) > 0 and lib.vln_top_logits_ws_bytes(0, 10, 0, 1) == 0

    def distill(bwd=False, **kw):
        a = L.Distill(p, 40, p, 3, p, 3, None, None, -1, p, p, 1.0, 1.0, 0, 0, 2, 40, 3, 0)
        for k, v in kw.items():
            if k not in ("red", "out", "ws", "g", "gs", "dz", "ldz"):
                setattr(a, k, v)
        if bwd:
            return lib.vln_distill_bwd(C.byref(a), kw.get("g", p), kw.get("gs", 0), None, kw.get("dz", p), kw.get("ldz", 40), None)
        return lib.vln_distill_fwd(C.byref(a), kw.get("red", 0), kw.get("out", None), kw.get("out", None), kw.get("ws", None), 0, None)

    for kw in (dict(N=0), dict(V=0), dict(logits=None), dict(ld=3), dict(K=0), dict(K=257, ld_ids=300, ld_teacher=300), dict(ids=None), dict(ld_ids=2), dict(type=2),
               dict(teacher_type=5), dict(temperature=0.0), dict(temperature=float("inf")), dict(alpha=0.5), dict(alpha=2.0, target=p), dict(rows=None),
               dict(stats=None), dict(red=1), dict(red=9, out=p), dict(V=1000000, ld=1000000)):
        assert distill(**kw) == 1, kw
        assert b"vln_distill_fwd" in lib.vln_last_error_string()
    for kw in (dict(g=None), dict(gs=2), dict(dz=None), dict(ldz=39)):
        assert distill(True, **kw) == 1, kw
    assert lib.vln_distill_fwd(None, 0, None, None, None, 0, None) == 1


def test_more_rows_than_a_launch_takes(vln):
    """A launch takes fewer than 2^32 threads along x and 65535 workgroups along y: refused before it, with a text."""
    lib, L = vln._lib.load(), vln._lib
    p = 4096
    a = L.Constrain()
    setattr(a, "in", p)
    a.out, a.ld_in, a.ld_out, a.B, a.V = p, 8, 8, 1 << 23, 8            # 512 threads a row
    assert lib.vln_constrain_logits(C.byref(a), None) == 1 and b"too many rows" in lib.vln_last_error_string()
    assert lib.vln_top_logits(p, 8, 0, 1 << 26, 8, 3, 1.0, p, p, p, None, 0, None) == 1 and b"too many" in lib.vln_last_error_string()
    assert lib.vln_top_logits(p, 1 << 30, 0, 1, (1 << 31) - 1, 3, 1.0, p, p, p, None, 0, None) == 1        # (ld < V)
    assert lib.vln_top_logits(p, 1 << 31, 0, 1, (1 << 31) - 1, 3, 1.0, p, p, p, None, 0, None) == 1 and b"too long rows" in lib.vln_last_error_string()
    d = L.Distill(p, 8, p, 3, p, 3, None, None, -1, p, p, 1.0, 1.0, 0, 0, 1 << 26, 8, 3, 0)                 # 64 threads a row
    assert lib.vln_distill_fwd(C.byref(d), 0, None, None, None, 0, None) == 1 and b"too many rows" in lib.vln_last_error_string()
