"""GPU: the word-logit operators where the speaker uses them -- decoding under constraints, a teacher's targets, the distillation loss in
teacher forcing and in the training iteration -- against plain restatements on the same modules."""
import numpy as np
import pytest
import torch

from conftest import load_golden
from parity import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
UNK, EOS, PAD = 1, 2, 0


@pytest.fixture(scope="module")
def vln():
    import vln_amd
    vln_amd._lib.load()
    return vln_amd


def make(vln, G, seed=None):
    cfg = G["cfg"]
    enc = vln.SpeakerEncoder(int(cfg["F"]), int(cfg["H"]), 0.5, True, int(cfg["ANG"]), 0.3)
    dec = vln.SpeakerDecoder(int(cfg["VOC"]), int(cfg["E"]), 0, int(cfg["H"]), 0.5)
    if seed is None:
        enc.load_state_dict(G["enc"], strict=True); dec.load_state_dict(G["dec"], strict=True)
    spk = vln.Speaker(enc.to(DEV), dec.to(DEV), max_decode=int(cfg["MAXD"]))
    enc.drop_ratio = enc.feat_drop_ratio = dec.drop_ratio = 0.0
    return spk


def inputs(G):
    return G["inp"]["can"].to(DEV), G["inp"]["img"].to(DEV), G["inp"]["lengths"].tolist()


def step_logits(vln, spk, can, img, lengths, fed):
    """[B, n, vocab] logits of a decoding loop that fed back the words `fed` [B, n] (the first word is <BOS>)."""
    from vln_amd.speaker import length2mask
    spk._mode(False)
    with torch.no_grad():
        ctx = spk.encoder(can.clone(), img.clone(), lengths)
        mask = length2mask(lengths, can.device, ctx.shape[1])
        words = torch.cat((torch.full((fed.shape[0], 1), spk.bos, dtype=torch.int64, device=DEV), fed[:, :-1]), 1)
        return spk.decoder(words, ctx, mask, *spk._zero_state(fed.shape[0], can.device))[0].double().cpu()


def constrained(z, words, mask, rep, pres, freq, bias):
    """One step's logits [B, V] under the constraints, in 64 bits; words: per row the ids so far."""
    out = z.clone()
    for b in range(z.shape[0]):
        for v in set(words[b]):
            c = words[b].count(v)
            x = out[b, v]
            out[b, v] = (x / rep if x > 0 else x * rep) - freq * c - pres
        for v, w in bias:
            out[b, v] += w
        out[b, ~mask[b]] = float("-inf")
        out[b, UNK] = float("-inf")
    return out


def test_decoding_under_constraints(vln):
    """Greedy decoding with penalties, biases and a grammar whose state alternates from word to word: every word is the largest of the
    constrained logits of the same modules on the words fed back, <UNK> never appears, and without constraints the words are the
    reference's as before."""
    G = load_golden("speaker_loop")
    spk = make(vln, G)
    can, img, lengths = inputs(G)
    V, B = int(G["cfg"]["VOC"]), can.shape[0]
    plain = spk.infer_batch(can.clone(), img.clone(), lengths)
    assert (plain == G["out"]["words_plain"].numpy()).all()
    states = torch.zeros(3, V, dtype=torch.bool)
    states[0, 2::2] = True                    # even words and <EOS>
    states[1, 3::2] = True
    states[1, EOS] = True
    states[2] = True
    fed = []

    def next_rows(t, words):
        assert words.shape == (B, t) and words.is_cuda
        fed.append(words.clone())
        rows = torch.full((B,), t % 2, dtype=torch.int64, device=DEV)
        rows[0] = 2 if t % 2 else -1          # one row is not constrained at all
        return rows

    cons = vln.vocab.WordConstraints(repetition=1.4, presence=0.3, frequency=0.2, bias_ids=torch.tensor([5, 8], device=DEV),
                                     bias_values=torch.tensor([0.75, -1.5], device=DEV), allowed=vln.vocab.pack_allowed(states).to(DEV), next_rows=next_rows)
    words = spk.infer_batch(can.clone(), img.clone(), lengths, constraints=cons)
    n = words.shape[1]
    # what was fed back: the model's own choice, also behind a row's <EOS> (the returned words are <PAD> there)
    chosen = torch.full((B, n), -1, dtype=torch.int64, device=DEV)
    for t in range(1, n):
        chosen[:, :t] = fed[t]
    live = torch.as_tensor(words) != PAD
    chosen[:, n - 1] = torch.where(live[:, n - 1], torch.as_tensor(words)[:, n - 1], torch.full((B,), 4)).to(DEV)
    assert torch.equal(chosen.cpu()[live], torch.as_tensor(words)[live]) and (words != UNK).all()
    z = step_logits(vln, spk, can, img, lengths, chosen)
    for t in range(n):
        mask = torch.stack([torch.ones(V, dtype=torch.bool) if b == 0 else states[t % 2] for b in range(B)])
        want = constrained(z[:, t], [chosen[b, :t].tolist() for b in range(B)], mask, 1.4, 0.3, 0.2, [(5, 0.75), (8, -1.5)])
        for b in range(B):
            if live[b, t]:
                # (the recomputed logits differ from the loop's by the recurrence's rounding: 1e-4 of their size, the modules' own bound)
                assert want[b, chosen[b, t]] >= want[b].max() - 2e-4 * want[b][torch.isfinite(want[b])].abs().max(), (b, t)
                assert torch.isfinite(want[b, chosen[b, t]])


def test_sampled_training_under_constraints(vln):
    """The speaker's own sampled training with constraints: the log-probabilities are those of the constrained distribution for the drawn
    words, and gradients reach the projection (0 for the banned words' rows)."""
    G = load_golden("speaker_loop")
    spk = make(vln, G)
    can, img, lengths = inputs(G)
    V, B = int(G["cfg"]["VOC"]), can.shape[0]
    ok = torch.ones(1, V, dtype=torch.bool)
    ok[0, 10:20] = False
    fed = []
    cons = vln.vocab.WordConstraints(repetition=1.5, frequency=0.3, allowed=vln.vocab.pack_allowed(ok).to(DEV),
                                     next_rows=lambda t, w: (fed.append(w.clone()), torch.zeros(B, dtype=torch.int64, device=DEV))[1])
    words, logp, _, ent = spk.infer_batch(can.clone(), img.clone(), lengths, sampling=True, train=True, constraints=cons)
    n = words.shape[1]
    assert (words != UNK).all() and not np.isin(words, np.arange(10, 20)).any()
    chosen = torch.as_tensor(words).to(DEV).clone()
    for t in range(1, n):
        chosen[:, :t] = fed[t]
    z = step_logits(vln, spk, can, img, lengths, chosen)
    live = torch.as_tensor(words) != PAD
    ref = torch.zeros(B, n, dtype=torch.float64)
    for t in range(n):
        s = constrained(z[:, t], [chosen[b, :t].tolist() for b in range(B)], ok.expand(B, V), 1.5, 0.0, 0.3, [])
        ref[:, t] = torch.log_softmax(s, 1).gather(1, chosen[:, t:t + 1].cpu()).view(-1)
    check(logp.detach().cpu()[live], ref[live], 2e-4, "log-probs of the sampled words")
    (logp.sum() + 0.1 * ent.sum()).backward()
    g = spk.decoder.projection.weight.grad
    assert torch.isfinite(g).all() and g.abs().sum() > 0 and (g[10:20] == 0).all() and (g[UNK] == 0).all()


def plain_distill(logits, targets, tgt, T, alpha, pad):
    """The loss on [N, V] logits in elementary operations (autograd does the rest)."""
    ids, tv, rest = targets
    u = torch.log_softmax(logits / T, 1)
    t = torch.cat((tv.double() / T, rest.double()[:, None]), 1)
    q = torch.softmax(t, 1)
    held = torch.zeros_like(logits, dtype=torch.bool).scatter_(1, ids, True)
    lrest = torch.logsumexp(u.masked_fill(held, float("-inf")), 1, keepdim=True)
    lp = torch.cat((u.gather(1, ids), lrest), 1)
    soft = (q * (torch.log(q) - lp)).sum(1)
    hard = -torch.log_softmax(logits, 1).gather(1, tgt[:, None]).view(-1)
    rows = alpha * T * T * soft + (1 - alpha) * hard
    live = tgt != pad
    return rows[live].mean()


def test_teacher_targets_and_distillation(vln):
    """A teacher's targets over one batch, and a student's distillation loss and gradients on them, against the plain formula on the
    student's own logits."""
    G = load_golden("speaker_loop")
    torch.manual_seed(5)
    teacher, student = make(vln, G), make(vln, G, seed=1)
    can, img, lengths = inputs(G)
    insts = G["inp"]["insts"].to(DEV)
    B, Lw = insts.shape
    T, alpha, k = 2.0, 0.7, 6
    targets = teacher.teacher_targets(can.clone(), img.clone(), lengths, insts, k, T, alpha)
    assert targets.ids.shape == (B * Lw, k) and not targets.values.requires_grad
    # the teacher's own logits, recomputed
    from vln_amd.speaker import length2mask
    with torch.no_grad():
        ctx = teacher.encoder(can.clone(), img.clone(), lengths)
        tz = teacher.decoder(insts, ctx, length2mask(lengths, can.device, ctx.shape[1]), *teacher._zero_state(B, can.device))[0].reshape(B * Lw, -1)
    sv, si = torch.sort(tz, dim=1, descending=True, stable=True)
    assert torch.equal(targets.ids, si[:, :k]) and torch.equal(targets.values, sv[:, :k])
    check(targets.rest, torch.logsumexp(sv[:, k:].double() / T, 1), 1e-6, "rest")
    with pytest.raises(ValueError):
        student.teacher_forcing(can.clone(), img.clone(), lengths, insts, train=False, distill=targets)
    loss = student.teacher_forcing(can.clone(), img.clone(), lengths, insts, train=True, distill=targets)
    loss.backward()
    grads = {p: p.grad.clone() for m in (student.encoder, student.decoder) for p in m.parameters() if p.grad is not None}
    for m in (student.encoder, student.decoder):
        m.zero_grad(set_to_none=True)
    student._mode(True)
    ctx = student.encoder(can.clone(), img.clone(), lengths)
    logits = student.decoder(insts, ctx, length2mask(lengths, can.device, ctx.shape[1]), *student._zero_state(B, can.device))[0].reshape(B * Lw, -1)
    tgt = torch.cat((insts[:, 1:], insts.new_zeros(B, 1)), 1).reshape(-1)
    ref = plain_distill(logits.double(), (targets.ids, targets.values, targets.rest), tgt, T, alpha, PAD)
    check(loss, ref, 1e-5, "loss")
    ref.backward()
    for m in (student.encoder, student.decoder):
        for n, p in m.named_parameters():
            if p.grad is not None:
                check(grads[p], p.grad, 1e-4, "grad " + n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distilling_iteration_as_one_graph_equals_eager(vln, dtype):
    """trainers.SpeakerIteration(distill=...): captured whole and replayed over changing batches and targets, losses and parameters equal the
    eager iterations' bit for bit."""
    dev = torch.device(DEV)
    B, Lp, Lw, V, F, vocab, k = 8, 4, 12, 36, 96, 50, 5

    def batch(i):
        g = torch.Generator().manual_seed(300 + i)
        lengths = torch.randint(2, Lp + 1, (B,), generator=g); lengths[0] = Lp
        insts = torch.randint(4, vocab, (B, Lw), generator=g); insts[:, 0] = 3
        insts[1, 7:] = 0
        t = torch.randn(B * Lw, vocab, generator=g) * 2
        tv, ids = torch.topk(t, k, dim=1)
        rest = torch.logsumexp(t.scatter(1, ids, float("-inf")) / 2.0, 1)
        return dict(can=(torch.randn(B, Lp, F, generator=g).abs() * 0.5).to(dev), img=(torch.randn(B, Lp, V, F, generator=g).abs() * 0.5).to(dev),
                    lengths=lengths, insts=insts.to(dev), teacher_ids=ids.to(dev), teacher_values=tv.to(dev), teacher_rest=rest.to(dev))

    runs = []
    for graph in (False, True):
        torch.manual_seed(29)
        it = vln.trainers.SpeakerIteration(dev, dtype, vocab=vocab, wemb=32, rnn=64, feature_size=F, angle_size=32, lr=1e-3, graph=True, distill=(2.0, 0.6))
        it.dec.deterministic_embedding_grad = True
        out = []
        it.load(batch(0))
        if graph:
            it.capture(warmup=3)
        else:
            for _ in range(3):
                it.iteration()
        for i in range(1, 5):
            it.load(batch(i))
            loss = it.replay() if graph else it.iteration()
            torch.cuda.synchronize()
            out.append((loss.detach().clone(), it.opt_e.flat_p.clone(), it.opt_d.flat_p.clone()))
        runs.append(out)
    for a, b in zip(*runs):
        assert torch.isfinite(a[0]).all() and all(torch.equal(x, y) for x, y in zip(a, b))
    assert not torch.equal(runs[0][0][0], runs[0][1][0])


def test_distilling_iteration_without_a_clock(vln):
    """The eager form on the caller's own batch, and targets that change the loss."""
    dev = torch.device(DEV)
    g = torch.Generator().manual_seed(1)
    B, Lp, Lw, V, F, vocab = 4, 3, 6, 36, 96, 50
    b = dict(can=(torch.randn(B, Lp, F, generator=g).abs()).to(dev), img=(torch.randn(B, Lp, V, F, generator=g).abs()).to(dev), lengths=torch.tensor([3, 3, 2, 1]),
             insts=torch.randint(4, vocab, (B, Lw), generator=g).to(dev), teacher_ids=torch.randint(0, vocab, (B * Lw, 3), generator=g).to(dev),
             teacher_values=torch.randn(B * Lw, 3, generator=g).to(dev))
    got = []
    for distill in (None, (1.0, 0.5)):
        torch.manual_seed(3)
        it = vln.trainers.SpeakerIteration(dev, torch.float32, vocab=vocab, wemb=32, rnn=64, feature_size=F, angle_size=32, distill=distill)
        got.append(float(it.iteration(b).detach()))
    assert np.isfinite(got).all() and got[0] != got[1]
