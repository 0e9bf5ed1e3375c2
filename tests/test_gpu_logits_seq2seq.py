"""The operators on output rows where the Seq2Seq model calls them: a teacher's top logits, a student's distillation loss, greedy
decode under constraints (sa_s2s_greedy_decode_constrained) against the same decode step by step."""
import math

import numpy as np
import pytest
import torch

from oracle import logits_ref as ref

pytestmark = pytest.mark.gpu

CFG = {"dropout": 0.0, "encoder": {"conv": [[8, 5, 11, 2]], "rnn": {"dim": 16, "bidirectional": True, "layers": 2}},
       "decoder": {"embedding_dim": 16, "layers": 1, "log_t": True}}
VOCAB = 14            # 12 letters, the end (12) and the start (13): K = 13 classes
END, START, K = 12, 13, 13


def build(seed, flatten=False):
    from speech_amd.models import Seq2Seq
    torch.manual_seed(seed)
    m = Seq2Seq(40, VOCAB, CFG).cuda()
    with torch.no_grad():
        m.fc.fc.weight.mul_(6)   # an untrained output is flat: answers that depend on the input
    if flatten:
        m.flatten_parameters_()
    return m


def batch(seed, B=5):
    rng = np.random.RandomState(seed)
    x = tuple(rng.randn(60 + 7 * b, 40).astype(np.float32) for b in range(B))
    y = tuple([START] + rng.randint(0, 12, 3 + b).tolist() + [END] for b in range(B))
    return x, y


def by_steps(m, b, max_len, states=None, next_states=None, **kw):
    """infer() token by token: decode_step, the restated constraints in 64 bits, the first maximum."""
    x, y = m.collate(*b)
    with torch.no_grad():
        enc = m.encode(x.cuda())
    B = enc.shape[0]
    tokens = y[:, :1].clone()
    state, cur = None, (states.cpu().clone() if states is not None else torch.zeros(B, dtype=torch.int32))
    for _ in range(max_len):
        out, state = m.decode_step(enc, tokens[:, -1:].cuda(), state=state)
        pen = {p: kw[p] for p in ("repetition", "presence", "frequency") if p in kw}
        other = {p: kw[p].cpu() for p in ("bias_ids", "bias_values", "mask") if p in kw}
        row = ref.constrain(out, history=tokens if pen else None, states=cur if "mask" in kw else None, **pen, **other)
        t = ref.pick(row)[0]
        t = torch.where(t < 0, END, t)
        if next_states is not None:
            n = next_states.cpu()
            cur = torch.tensor([int(n[s, v]) if 0 <= s < n.shape[0] else int(s) for s, v in zip(cur.tolist(), t.tolist())]).int()
        tokens = torch.cat([tokens, t[:, None]], 1)
        if bool((t == END).all()):
            break
    return tokens.tolist()


def grammar(seed, S=6):
    """Each state allows some letters and leads on; the last one allows the end alone and stays."""
    from speech_amd.logits import pack_mask
    g = torch.Generator().manual_seed(seed)
    allowed = torch.rand(S, K, generator=g) < 0.4
    allowed[:, 3] = True
    allowed[S - 1] = False
    allowed[S - 1, END] = True
    following = (torch.arange(S)[:, None] + 1 + torch.randint(0, 2, (S, K), generator=g)).clamp(max=S - 1).int()
    return pack_mask(allowed).cuda(), following.cuda(), allowed


def test_neutral_constraints_change_nothing():
    m = build(1)
    m.set_eval()
    for seed in range(3):
        b = batch(seed)
        want = m.infer(b, max_len=14)
        assert m.infer(b, max_len=14, constraints={}) == want
        assert m.infer(b, max_len=14, constraints=dict(repetition=1.0, presence=0.0)) == want
        mask = torch.full((2, 1), -1, dtype=torch.int32).cuda()
        assert m.infer(b, max_len=14, constraints=dict(mask=mask)) == want


@pytest.mark.parametrize("case", ["penalties", "per_request", "bias", "grammar", "all", "states"])
def test_constrained_infer_against_the_steps(case):
    m = build(2)
    m.set_eval()
    B = 5
    g = torch.Generator().manual_seed(3)
    mask, following, _ = grammar(5)
    kw = {}
    if case in ("penalties", "all"):
        kw.update(repetition=1.7, presence=0.6, frequency=0.3)
    if case == "per_request":
        kw.update(repetition=(torch.rand(B, generator=g) + 1).cuda(), frequency=torch.rand(B, generator=g).cuda())
    if case in ("bias", "all"):
        kw.update(bias_ids=torch.randint(0, K, (B, 4), generator=g).cuda(), bias_values=(torch.randn(B, 4, generator=g) * 4).cuda())
    if case in ("grammar", "all", "states"):
        kw.update(mask=mask, next_states=following)
    if case == "states":
        kw["states"] = torch.tensor([0, -1, 3, 6, 5], dtype=torch.int32).cuda()   # -1 and 6: no grammar
    start = kw["states"].clone() if "states" in kw else None
    for seed in range(4):
        b = batch(seed, B)
        assert m.infer(b, max_len=12, constraints=kw) == by_steps(m, b, 12, **kw), (case, seed)
    if start is not None:
        assert torch.equal(kw["states"], start)   # the caller's states are not moved on


def test_constrained_answers_obey_the_grammar_and_end_where_nothing_is_left():
    from speech_amd.logits import pack_mask
    m = build(4)
    m.set_eval()
    mask, following, allowed = grammar(7)
    for tokens in m.infer(batch(9), max_len=20, constraints=dict(mask=mask, next_states=following)):
        s = 0
        for t in tokens[1:]:
            assert bool(allowed[s, t])
            s = int(following[s, t])
        assert tokens[-1] == END
    nothing = pack_mask(torch.zeros(1, K, dtype=torch.bool)).cuda()
    assert m.infer(batch(9), max_len=20, constraints=dict(mask=nothing)) == [[START, END]] * 5


def test_constrained_infer_never_answers_nan():
    """A token whose constrained logit is NaN is passed over, like one that is banned; with nothing else left the request ends."""
    m = build(4)
    m.set_eval()
    g = torch.Generator().manual_seed(12)
    ids = torch.stack([torch.randperm(K, generator=g)[:5] for _ in range(5)]).cuda()
    b = batch(3)
    def answers(value):
        return m.infer(b, max_len=12, constraints=dict(bias_ids=ids, bias_values=torch.full((5, 5), value).cuda()))
    assert answers(math.nan) == answers(-math.inf)
    every = torch.arange(K).repeat(5, 1).cuda()
    nan = torch.full((5, K), math.nan).cuda()
    assert m.infer(b, max_len=12, constraints=dict(bias_ids=every, bias_values=nan)) == [[START, END]] * 5


def test_constrained_infer_refuses():
    from speech_amd._lib import SpeechAmdError
    m = build(5)
    m.set_eval()
    b = batch(1)
    mask, following, _ = grammar(7)
    for kw in (dict(next_states=following), dict(mask=mask, next_states=following.long()), dict(mask=mask, next_states=following[:, :5]),
               dict(mask=mask, states=torch.zeros(4, dtype=torch.int32).cuda()), dict(mask=mask.cpu()), dict(repetition=0.0),
               dict(bias_ids=torch.zeros(5, 2, dtype=torch.int64).cuda())):
        with pytest.raises(SpeechAmdError):
            m.infer(b, max_len=4, constraints=kw)
    with pytest.raises(TypeError):
        m.infer(b, max_len=4, constraints=dict(history=torch.zeros(5, 2, dtype=torch.int64).cuda()))


def same(name, got, want, rel):
    """Parameter gradients that come from nearly the same logits' gradients through the same decoder backward."""
    if name == "attend.nn.1.fc.bias":
        # it shifts every score of a softmax, so its gradient is 0 and what is there are roundings: some 1100 terms (5 utterances, 8
        # tokens, 28 frames) whose absolute values sum to no more than 40 tokens * 2 * 0.05 * log(28) = 13, summed in any order:
        # 1100 * 2^-24 * 13 = 9e-4
        assert float(got.abs().max()) <= 1e-3 and float(want.abs().max()) <= 1e-3
        return
    assert float((got - want).abs().max()) <= rel * max(float(want.abs().max()), 1e-3), name


@pytest.mark.parametrize("flatten", [False, True])
def test_distillation_of_one_model_into_another(flatten):
    """Teacher -> top_logits -> distill_loss: at alpha = 0 it is loss(), with the teacher's own weights the soft part and its
    gradient vanish, and elsewhere value and parameter gradients are those of the definition through autograd."""
    from speech_amd import ops
    teacher, student = build(6), build(7, flatten)
    teacher.set_eval()
    student.set_train()
    b = batch(2)
    k, T = 5, 2.0
    values, ids, rest = teacher.top_logits(b, k, T)
    U1 = max(len(l) for l in b[1]) - 1
    assert values.shape == ids.shape == (5, U1, k) and rest.shape == (5, U1)
    with torch.no_grad():
        wv, wi, wr = ref.top_logits(teacher(b), k, T)
    assert torch.equal(ids.cpu(), wi) and torch.equal(values.cpu().double(), wv)

    def grads(loss):
        student.zero_grad(set_to_none=True)
        ops.backward(loss)
        return {n: (p._grad_slot if flatten else p.grad).detach().clone() for n, p in student.named_parameters()}

    # alpha = 0 is loss(): both are float32 sums of the same numbers, in another order
    plain = student.loss(b)
    hard = student.distill_loss(b, values, ids, rest, temperature=T, alpha=0.0)
    assert abs(float(plain.detach()) - float(hard.detach())) <= 64 * 2.0 ** -24 * abs(float(plain.detach()))
    a, c = grads(student.loss(b)), grads(hard)
    for n in a:
        same(n, c[n], a[n], 1e-5)
    # the definition: the gradient of the logits in 64 bits, through the same decoder backward
    for alpha, tail in ((0.6, rest), (1.0, None)):
        w = torch.ones(5, U1)
        w[1, 2:] = 0.0
        loss = student.distill_loss(b, values, ids, tail, weights=w.cuda(), temperature=T, alpha=alpha)
        got = grads(loss)
        x, y = student.collate(*b)
        out, _ = student.forward_impl(x.cuda(), y.cuda())
        wl, wg, _ = ref.distill(out, values, ids, rest=tail, targets=y[:, 1:], weights=w, temperature=T, alpha=alpha, denom=5)
        assert abs(float(loss.detach()) - float(wl)) <= 1e-5 * abs(float(wl))
        student.zero_grad(set_to_none=True)
        out.backward(gradient=wg.float().cuda())
        for n, p in student.named_parameters():
            same(n, got[n], (p._grad_slot if flatten else p.grad).detach(), 1e-4)
    # its own teacher: KL of a distribution with itself
    student.set_eval()
    own = student.top_logits(b, k, T)
    student.set_train()
    loss = student.distill_loss(b, *own, temperature=T, alpha=1.0)
    rows = 5 * U1
    assert abs(float(loss.detach())) <= rows / 5 * T * T * 200 * 2.0 ** -24
    assert max(float(v.abs().max()) for v in grads(loss).values()) < 1e-3


def test_a_teacher_in_training_mode_reads_the_labels():
    """Dropout and scheduled sampling are the model's own training: the rows it teaches belong to the labels, and both are on again
    afterwards, also when the call fails."""
    from speech_amd._lib import SpeechAmdError
    from speech_amd.models import Seq2Seq
    cfg = {"dropout": 0.5, "encoder": CFG["encoder"], "decoder": dict(CFG["decoder"], sample_prob=0.5)}
    torch.manual_seed(10)
    m = Seq2Seq(40, VOCAB, cfg).cuda()
    b = batch(6)
    m.set_eval()
    want = m.top_logits(b, 5, 2.0)
    assert not m.training and not m.scheduled_sampling and m.volatile
    m.set_train()
    m.attend.eval()
    for _ in range(3):
        got = m.top_logits(b, 5, 2.0)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        assert m.training and m.scheduled_sampling and not m.volatile
        assert not m.attend.training and not m.attend.conv.training and m.dec_rnn.training
    with pytest.raises(SpeechAmdError):
        m.top_logits(b, K + 1)
    assert m.training and m.scheduled_sampling


def test_teach_train_and_answer():
    """One small run of all of it: a few steps on a teacher's top logits, then answers under a grammar and penalties."""
    from speech_amd import ops
    teacher, student = build(8), build(9, True)
    teacher.set_eval()
    student.set_train()
    b = batch(4)
    top = teacher.top_logits(b, 6, 2.0)
    params, flat = student._flat
    for _ in range(5):
        student.zero_grad(set_to_none=True)
        loss = student.distill_loss(b, *top, temperature=2.0, alpha=0.7)
        ops.backward(loss)
        ops.stamp_health(flat)
        ops.clip_sgd_step(params, flat, None, 1e-3, 0.0, 200.0)
        assert math.isfinite(float(loss.detach()))
    student.set_eval()
    mask, following, _ = grammar(11)
    out = student.infer(b, max_len=10, constraints=dict(mask=mask, next_states=following, repetition=1.2, frequency=0.1))
    assert len(out) == 5 and all(t[0] == START and t[-1] == END for t in out)
