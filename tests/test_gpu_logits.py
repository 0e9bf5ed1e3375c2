"""speech_amd.logits on the GPU against the restatement in 64 bits (oracle/logits_ref.py).

Tolerances, u = 2^-24 (half a step of float32), E = half a step of the logits' type (2^-24, 2^-8, 2^-11):
  * constrained logits: at most six roundings of numbers no larger than |x| max(r, 1/r) + c f + p + |b|, then one to the type.
  * log-sum-exps: x - m is rounded once, times log2(e) / T twice more: 3 u |x - m| / T in a term's exponent; exp2 itself and a sum
    of depth <= 40 (lanes, waves, segments) add 42 u; the logarithm and the final sum one u of their value each.
  * gradients: coefficient * (p, q, p1, 1) with those relative errors, then one rounding to the type and, where the result is
    subnormal, half its smallest step."""
import math

import numpy as np
import pytest
import torch

from oracle import logits_ref as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}  # results below are flushed / half a step
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def L():
    from speech_amd import logits
    return logits


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def rows_like(g, n, V, dtype):
    x = torch.randn(n, V, generator=g) * 2
    x[torch.rand(n, V, generator=g) < 0.01] += 6
    return x.to(dtype)


def cuda(d):
    return {k: v.cuda() if torch.is_tensor(v) else v for k, v in d.items()}


def constraints(g, n, V, length, biases, grammar, scalars=False):
    kw = {}
    if length is not None:
        kw["history"] = torch.randint(-2, max(1, min(V, length // 3 + 1)) + 2, (n, length), generator=g)  # repeats; some are no class
        kw["lengths"] = torch.randint(-1, length + 3, (n,), generator=g).int()                            # some beyond the row
        if scalars:
            kw.update(repetition=1.3, presence=0.4, frequency=0.15)
        else:
            kw.update(repetition=torch.rand(n, generator=g) + 0.7, presence=torch.rand(n, generator=g) - 0.3,
                      frequency=torch.rand(n, generator=g) * 0.3)
    if biases:
        kw["bias_ids"] = torch.randint(-1, V + 1, (n, biases), generator=g)   # duplicates where V is small; some are no class
        kw["bias_values"] = torch.randn(n, biases, generator=g) * 3
    if grammar:
        S = 5
        allowed = torch.rand(S, V, generator=g) < 0.6
        allowed[:, 0] = True
        kw["mask"] = L().pack_mask(allowed)
        kw["states"] = (torch.arange(n) % (S + 2) - 1).int()                  # -1 and S: no grammar
    return kw


SHAPES = [(1, 1, 0, 0, True), (2, 29, 40, 3, True), (32, 29, 200, 0, True), (3, 32, 7, 50, False), (5, 1000, None, 9, True),
          (3, 4095, 300, 20, True), (2, 4096, 5000, 0, False), (4, 4097, 64, 64, True), (3, 8193, 600, 10, True), (2, 16385, 1, 1, True),
          (2, 32000, 1500, 128, True), (7, 50021, 333, 16, True), (2, 131072, 4096, 100, True), (1, 262147, 70, 5, False),
          (1, 1048576, 900, 300, True), (1, 1044481, 64, 0, False), (130, 8190, 20, 2, True),
          (600, 8190, 9, 3, True),
          # long lists and enough rows for larger workgroups; one entry too few for them
          (800, 5000, 1100, 40, True), (160, 40003, 3000, 0, False), (258, 16385, 1000, 25, True), (258, 16385, 1000, 24, True)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,V,length,biases,grammar", SHAPES)
def test_constrain_and_pick(n, V, length, biases, grammar, dtype):
    g = gen(n * 7 + V)
    x = rows_like(g, n, V, dtype)
    kw = constraints(g, n, V, length, biases, grammar, scalars=n == 3)
    want = ref.constrain(x, **kw)
    got = L().constrain(x.cuda(), **cuda(kw))
    assert got.dtype == dtype and got.shape == x.shape
    got = got.cpu().double()
    assert torch.equal(got == -math.inf, want == -math.inf)
    big = x.double().abs() * 1.7 + (length or 0) * 0.3 + 1 + (15 if biases else 0)
    fine = want > -math.inf
    touched = 6 * U * big + HALF[dtype] * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert bool(((got - want).abs() <= touched)[fine].all())
    if length is None and not biases:
        assert torch.equal(got[fine], x.double()[fine])
    tokens, logp = L().pick(x.cuda(), **cuda(kw))
    assert tokens.dtype == torch.int64 and logp.dtype == torch.float32
    wt, wl = ref.pick(want)
    tokens = tokens.cpu()
    at = want.gather(1, tokens[:, None])[:, 0]  # a near tie may fall either way by the roundings of the two values
    assert bool((want.gather(1, wt[:, None])[:, 0] - at <= 12 * U * float(big.max())).all())
    same = tokens == wt
    assert bool(same.float().mean() > 0.5)
    spread = float((want.max(1, keepdim=True).values - want)[fine].max())
    tol = (3 * spread + 42 + 12 * float(big.max())) * U + 2 * U * wl.abs()
    assert bool(((logp.cpu().double() - wl).abs() <= tol).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [29, 5000, 40000])
def test_pick_ties_go_to_the_lowest_token(V, dtype):
    """Quarters and powers of two: every step is exact, ties are real ties."""
    g = gen(V)
    n = 24
    x = (torch.randint(-8, 9, (n, V), generator=g) / 4).to(dtype)
    kw = dict(history=torch.randint(0, V, (n, 50), generator=g), repetition=2.0, presence=0.5, frequency=0.25,
              bias_ids=torch.randint(0, V, (n, 6), generator=g), bias_values=torch.randint(0, 3, (n, 6), generator=g) / 4,
              mask=L().pack_mask(torch.rand(n, V, generator=g) < 0.7))
    want = ref.constrain(x, **kw)
    assert torch.equal(L().constrain(x.float().cuda(), **cuda(kw)).cpu().double(), want)
    tokens, _ = L().pick(x.cuda(), **cuda(kw))
    assert torch.equal(tokens.cpu(), ref.pick(want)[0])


def test_pick_of_rows_that_are_not_ordinary():
    V = 10000
    x = torch.zeros(9, V)
    x[0] = -math.inf                              # nothing is left
    x[1, 77] = math.nan
    x[1, 99] = math.nan
    x[2, 5000] = math.inf
    x[3, [4000, 9000]] = math.inf                 # two forced tokens: half each
    x[4] = torch.finfo(torch.float32).min         # the type's lowest value is a value
    x[5] = -math.inf
    x[5, V - 1] = -3.0
    x[6] = -0.0
    x[6, 3] = 0.0                                 # equal to -0: the lowest token
    x[7, 11] = math.nan                           # masked below
    x[8, 12] = 5.0
    allowed = torch.ones(9, V, dtype=torch.bool)
    allowed[7, 11] = False
    allowed[8] = False
    kw = dict(mask=L().pack_mask(allowed).cuda())
    tokens, logp = L().pick(x.cuda(), **kw)
    assert tokens.tolist() == [-1, 77, 5000, 4000, 0, V - 1, 0, 0, -1]
    logp = logp.cpu().double()
    assert logp[0] == logp[8] == -math.inf and logp[1].isnan() and logp[2] == logp[5] == 0.0
    for b, want in ((3, -math.log(2)), (4, -math.log(V)), (6, -math.log(V)), (7, -math.log(V - 1))):
        assert abs(float(logp[b]) - want) <= 44 * U + 2 * U * abs(want), b
    y = L().constrain(x.cuda(), **kw).cpu()
    assert bool((y[8] == -math.inf).all()) and y[7, 11] == -math.inf and y[1, 77].isnan()
    # a bias of +inf forces its token, one of -inf bans it
    ids = torch.tensor([[5, 6]]).cuda()
    tokens, logp = L().pick(torch.zeros(1, 10).cuda(), bias_ids=ids, bias_values=torch.tensor([[-math.inf, math.inf]]).cuda())
    assert tokens.tolist() == [6] and logp.tolist() == [0.0]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V,ld,off", [(29, 31, 1), (4097, 4100, 3), (20001, 20004, 5), (20000, 20008, 0)])
def test_constrain_in_place_on_rows_with_gaps(V, ld, off, dtype):
    g = gen(V)
    n = 5
    flat = rows_like(g, 1, off + n * ld + 16, dtype)[0]
    kw = constraints(g, n, V, 60, 12, True)
    dev = flat.cuda()
    x = dev[off:off + n * ld].view(n, ld)[:, :V]
    want = L().constrain(x.contiguous(), **cuda(kw))
    out = L().constrain(x, out=x, **cuda(kw))
    assert out.data_ptr() == x.data_ptr() and torch.equal(x, want)
    keep = torch.ones(flat.numel(), dtype=torch.bool)  # what lies between, before and behind the rows is as it was
    keep[off:off + n * ld].view(n, ld)[:, :V] = False
    assert torch.equal(dev.cpu()[keep], flat[keep])
    other = torch.empty(n, ld + 3, dtype=dtype, device="cuda")[:, 3:3 + V]   # another alignment than the input's
    y = flat.cuda()[off:off + n * ld].view(n, ld)[:, :V]
    assert torch.equal(L().constrain(y, out=other, **cuda(kw)), want)
    (ta, la), (tb, lb) = L().pick(y, **cuda(kw)), L().pick(y.contiguous(), **cuda(kw))
    assert torch.equal(ta, tb)
    # the sum runs in another order where a row starts at another offset from a 16-byte boundary: each side is within the
    # tolerance of a log-sum-exp (top of this file; |x - m| < 60 here) of the same number, so they are within twice that
    assert float((la - lb).abs().max()) <= 2 * ((3 * 60 + 42) * U + 2 * U * float(la.abs().max()))


def test_lists_and_masks_that_are_views():
    """Histories, bias lists and masks as stretches of wider tensors (a token matrix that is still being written, ...)."""
    g = gen(33)
    n, V = 6, 5003
    x = rows_like(g, n, V, torch.float32)
    kw = constraints(g, n, V, 60, 9, True)
    want = ref.constrain(x, **kw)
    wide = dict(kw)
    for name, pad in (("history", 11), ("bias_ids", 4), ("bias_values", 4), ("mask", 3)):
        t = torch.randint(0, 9, (kw[name].shape[0], kw[name].shape[1] + 2 * pad), generator=g).to(kw[name].dtype)
        t[:, pad:-pad] = kw[name]
        wide[name] = t.cuda()[:, pad:-pad]
    got = L().constrain(x.cuda(), **cuda(wide))
    assert torch.equal(got, L().constrain(x.cuda(), **cuda(kw)))
    assert torch.equal(L().pick(x.cuda(), **cuda(wide))[0].cpu(), ref.pick(want)[0])


def test_constrain_refuses_on_the_gpu():
    from speech_amd._lib import SpeechAmdError
    x = torch.zeros(3, 40).cuda()
    for kw in (dict(history=torch.zeros(3, 4, dtype=torch.int64)), dict(out=torch.zeros(3, 41).cuda()),
               dict(out=torch.zeros(3, 40).cuda().half()), dict(out=torch.zeros(3, 40)),
               dict(out=torch.zeros(1, 40).cuda().expand(3, 40)), dict(out=torch.zeros(3, 40).cuda().requires_grad_())):
        with pytest.raises(SpeechAmdError):
            L().constrain(x, **kw)
    wide = torch.zeros(4, 80).cuda()
    with pytest.raises(SpeechAmdError, match="share"):
        L().constrain(wide[:3], out=wide[1:])
    L().constrain(wide[:, :40], bias_ids=torch.zeros(4, 1, dtype=torch.int64).cuda(), bias_values=torch.ones(4, 1).cuda(), out=wide[:, 40:])
    assert wide[:, 40].tolist() == [1.0] * 4 and float(wide.abs().sum()) == 4.0
    with pytest.raises(SpeechAmdError):
        L().pick(torch.zeros(2, 3, 40).cuda())
    seen = x._version   # written in place: whoever saved the tensor must see that
    L().constrain(x, out=x)
    assert x._version > seen
    assert L().constrain(x[:0]).shape == (0, 40) and L().pick(x[:0])[0].shape == (0,)


def test_a_batch_without_requests():
    x = torch.zeros(0, 40).cuda()
    none = torch.zeros(0, 5, dtype=torch.int64).cuda()
    kw = dict(history=none, lengths=torch.zeros(0, dtype=torch.int32).cuda(), frequency=0.5, bias_ids=none, bias_values=torch.zeros(0, 5).cuda(),
              mask=torch.zeros(0, 2, dtype=torch.int32).cuda())
    assert L().constrain(x, **kw).shape == (0, 40)
    tokens, logp = L().pick(x, **kw)
    assert tokens.shape == logp.shape == (0,)


# ---- top_logits ----------------------------------------------------------------------------------------------------------
def check_top(x, k, temperature=1.0, got=None):
    values, ids, rest = L().top_logits(x.cuda(), k, temperature) if got is None else got
    wv, wi, wr = ref.top_logits(x, k, temperature)
    assert values.dtype == rest.dtype == torch.float32 and ids.dtype == torch.int64
    assert torch.equal(ids.cpu(), wi)
    assert torch.equal(values.cpu().double().nan_to_num(nan=1e300), wv.nan_to_num(nan=1e300))
    got = rest.cpu().double()
    fine = wr.isfinite()
    assert torch.equal(got[~fine].nan_to_num(nan=1e300), wr[~fine].nan_to_num(nan=1e300))
    d = x.double()
    d = torch.where(d.isfinite(), d, 0.0)
    tol = (3 * float(d.max() - d.min()) / temperature + 42) * U + 3 * U * wr.abs() + 2 * U * float(d.abs().max()) / temperature
    assert bool(((got - wr).abs() <= tol)[fine].all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,V,k", [(1, 1, 1), (5, 2, 2), (40, 29, 8), (700, 29, 29), (9, 64, 5), (9, 65, 33), (6, 128, 128), (3, 129, 128),
                                   (4, 511, 20), (4, 1000, 64), (3, 4099, 100), (2, 8192, 1), (2, 8195, 128), (3, 32000, 64),
                                   (2, 50021, 100), (3, 131071, 128), (1, 300007, 50),
                                   (1, 1048576, 128), (1, 1044483, 20),
                                   # enough rows for a wave each, for a workgroup each, and just too few
                                   (1100, 131, 5), (1024, 257, 128), (1030, 1000, 64), (1100, 1021, 100), (1023, 1000, 64), (1040, 2003, 33),
                                   (260, 8200, 20), (256, 20000, 64), (255, 20000, 64), (257, 32768, 128), (258, 33001, 7)])
def test_top_logits(n, V, k, dtype):
    check_top(rows_like(gen(V + k), n, V, dtype), k, 1.0 if n % 2 else 2.5)


@pytest.mark.parametrize("V,times", [(29, 1), (300, 1), (5000, 1), (40000, 1), (300, 74), (1000, 74), (9000, 19), (30000, 19)])
@pytest.mark.parametrize("k", [1, 20, 128])
def test_top_logits_of_rows_that_are_not_ordinary(V, times, k):
    k = min(k, V)
    g = gen(V * k)
    x = torch.randn(14, V, generator=g)
    x[0] = 1.5                                               # all equal: the lowest ids
    x[1] = torch.arange(V).float()                           # ascending
    x[2] = -torch.arange(V).float()                          # descending
    x[3] = -math.inf
    x[4, ::2] = -math.inf
    x[5] = torch.finfo(torch.float32).min
    x[6, V // 2] = math.nan
    x[7] = math.nan
    x[8, [0, V - 1]] = math.inf
    x[9] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)   # equal: the lowest ids, whatever the sign
    x[10, :min(V, 400)] += 50                                # all of the top in one stretch
    x[11, 4::max(1, V // 37)] += 50                          # ... at one step
    x[12] = torch.randint(0, 3, (V,), generator=g).float()   # many ties
    x[13] = -x[13].abs() - 100
    for dtype in TYPES:
        y = x.to(dtype)
        if times == 1:
            check_top(y, k, 1.0)
            continue
        many = L().top_logits(y.cuda().repeat(times, 1), k)   # other launch shapes; every copy of a row has the same answer
        many = [t.view(times, 14, *t.shape[1:]) for t in many]
        for t in many:
            bits = t.view(torch.int32) if t.dtype == torch.float32 else t
            assert bool((bits == bits[:1]).all())
        check_top(y, k, 1.0, got=[t[0] for t in many])


@pytest.mark.parametrize("V,times", [(29, 1), (300, 1), (5000, 1), (40000, 1), (300, 86), (1000, 86), (9000, 22), (30000, 22)])
@pytest.mark.parametrize("k", [1, 20, 128])
def test_the_rest_of_rows_that_are_not_ordinary(V, times, k):
    """Like the rows above, each held to the tolerance of its own range: where all of the top lies in one stretch or at one step, many
    ties, all equal, a second stretch far below, a slope."""
    k = min(k, V)
    g = gen(V * k + 1)
    x = torch.randn(12, V, generator=g)
    x[0] = 1.5
    x[1] = torch.arange(V).float() * (20.0 / V)
    x[2] = -torch.arange(V).float() * (20.0 / V)
    x[3, ::2] = -math.inf
    x[4, [0, V - 1]] = math.inf
    x[5] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)
    x[6, :min(V, 400)] += 50
    x[7, 4::max(1, V // 37)] += 50
    x[8] = torch.randint(0, 3, (V,), generator=g).float()
    x[9] = -x[9].abs() - 100
    x[10, V // 2:] -= 30
    x[11] *= 5
    for dtype in TYPES:
        y = x.to(dtype)
        many = L().top_logits(y.cuda().repeat(times, 1), k)
        many = [t.view(times, 12, *t.shape[1:])[0] for t in many]
        for row in range(12):
            check_top(y[row:row + 1], k, 1.0, got=[t[row:row + 1] for t in many])
    low = torch.full((3, V), torch.finfo(torch.float32).min)   # the type's lowest value is a number: rest = it + log(V - k) = it
    rest = L().top_logits(low.cuda(), k)[2]
    want = low[0, 0] if V > k else torch.tensor(-math.inf)
    assert bool((rest.cpu() == want).all())


@pytest.mark.parametrize("V,times", [(129, 1), (700, 1), (1000, 64), (9000, 16), (30000, 16), (40000, 1), (200001, 1)])
@pytest.mark.parametrize("k", [5, 128])
def test_top_logits_of_masked_rows(V, times, k):
    """A mask that leaves fewer than k, exactly k, a few more or many more, at both ends and between; NaN in many places."""
    g = gen(V + k)
    kept = [0, 1, k - 1, k, k + 1, k + 40, 2 * k + 200]
    rows = []
    for fill in (-math.inf, -60000.0, 0.0):
        for n in kept:
            x = torch.full((V,), fill)
            at = torch.randperm(V, generator=g)[:n] if n % 2 else torch.arange(V)[-n:] if n else torch.arange(0)
            x[at] = torch.randn(len(at), generator=g) * 3 + (5 if fill == 0.0 else 0)
            rows.append(x)
    for n in (k // 2 + 1, min(V, 300), min(V, 2 * k + 300)):
        x = torch.randn(V, generator=g)
        x[torch.randperm(V, generator=g)[:n]] = math.nan
        rows.append(x)
    x = torch.stack(rows)
    for dtype in TYPES:
        y = x.to(dtype)
        got = L().top_logits(y.cuda().repeat(times, 1), k)
        got = [t.view(times, len(rows), *t.shape[1:]) for t in got]
        for t in got:
            bits = t.view(torch.int32) if t.dtype == torch.float32 else t
            assert bool((bits == bits[:1]).all())
        for i in range(len(rows)):  # (one at a time: the tolerance is that of a row's own range)
            check_top(y[i:i + 1], k, 1.0, got=[t[0, i:i + 1] for t in got])


@pytest.mark.parametrize("V", [9001, 40000, 200001])
def test_top_logits_where_the_others_lie_far_below(V):
    """The k-th value is far above everything that is left, in the whole row or in one stretch of it only."""
    g = gen(V)
    k = 64
    x = torch.randn(6, V, generator=g)
    x[0, torch.randperm(V, generator=g)[:k]] += 60
    x[1, torch.randperm(V, generator=g)[:k]] += 3000
    x[2, :] = -1e30
    x[2, torch.randperm(V, generator=g)[:k]] = 5.0
    x[3, : V // 3] -= 50                                       # one third holds ties at the top and nothing near them
    x[3, torch.randperm(V // 3, generator=g)[:k]] = 10.0
    x[3, V // 3:] -= 25
    x[4] = -math.inf
    x[4, torch.randperm(V, generator=g)[:k + 1]] = torch.randn(k + 1, generator=g) * 30
    x[5, torch.randperm(V, generator=g)[:k + 40]] += 45
    for dtype in (torch.float32, torch.bfloat16):
        for row in range(6):
            check_top(x[row:row + 1].to(dtype), k, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("n,V", [(1100, 900), (600, 1000), (600, 2000), (300, 4000), (300, 8000), (300, 16000), (260, 32000), (40, 40000),
                                 (3, 300007)])
def test_top_logits_that_stand_out_in_every_kernel_form(n, V, dtype):
    """A few more than k tokens stand out and the others vanish beside them: the candidates fit at once, and the row is looked at again
    for the others' sum alone.  Every form of the kernel (a wave, 256 to 1024 threads, segments), the top scattered or in one stretch;
    the lists and the bits of every run are the same."""
    g = gen(n + V)
    k = 40
    for fill in (-math.inf, -200.0):
        x = torch.full((n, V), fill)
        for b in range(n):
            many = k + 7 * (b % 5)
            at = torch.randperm(V, generator=g)[:many] if b % 2 else torch.randint(0, V - 2 * k, (1,), generator=g) + torch.randperm(2 * k, generator=g)[:many]
            x[b, at] = torch.randn(many, generator=g) * 3 + 50
        x = x.to(dtype)
        dev = x.cuda()
        want = L().top_logits(dev, k)
        check_top(x, k, got=want)
        for _ in range(4):
            assert all(torch.equal(a, b) for a, b in zip(L().top_logits(dev, k), want))


@pytest.mark.parametrize("n,V,k", [(8, 131071, 100), (2, 300007, 128), (1, 1048576, 128)])
def test_top_logits_with_a_long_list_of_small_terms(n, V, k):
    """One token of the others stands at 0 and thousands at -22.4, below 2^-32 of it each, in the lists that long rows are joined from:
    together they are up to 70 * 2^-24 of the sum.  The sum S is 1 and a little: each of the two roundings of a float32 sum there is half
    a step of [1, 2), 2^-24; log(S) and the small terms themselves are off by less than 2^-24 of a few 2^-19; in all 4 * 2^-24."""
    g = gen(V)
    x = torch.full((n, V), -40.0)
    step = 7000                                       # less than any segment of such rows
    for b in range(n):
        for at in range(0, V - step + 1, step):
            x[b, at + torch.randperm(step, generator=g)[:150]] = -22.4
        at = torch.randperm(step, generator=g)[:k + 1]
        x[b, at[:k]] = 10.0 + torch.arange(k) / 16
        x[b, at[k]] = 0.0
    _, ids, rest = L().top_logits(x.cuda(), k)
    _, wi, wr = ref.top_logits(x, k)
    assert torch.equal(ids.cpu(), wi)
    assert float((wr - (x == -22.4).sum(1) * math.exp(-22.4)).abs().max()) < 1e-8    # (the list is what counts beside the 1)
    assert float((rest.cpu().double() - wr).abs().max()) <= 4 * U


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [29, 5001, 33000])
def test_top_logits_of_views(V, dtype):
    """Time-major rows handed over batch-first, rows with gaps, rows at odd offsets: read in place."""
    g = gen(V)
    T, B = 6, 3
    base = rows_like(g, T * B, V + 3, dtype).view(T, B, V + 3)
    x = base.cuda().transpose(0, 1)[..., 1:V + 1]
    got = L().top_logits(x, 7)
    want = L().top_logits(x.contiguous(), 7)
    assert got[0].shape == (B, T, 7) and got[2].shape == (B, T)
    # the list is the same in every layout; the sum of the others runs in another order where a row starts at another offset
    # from a 16-byte boundary, so each side is within the tolerance of a log-sum-exp (top of this file) and not within bits
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    plain = base.transpose(0, 1)[..., 1:V + 1]
    check_top(plain, 7, got=got)
    check_top(plain, 7, got=want)
    assert L().top_logits(x[:, :0], 7)[0].shape == (B, 0, 7)


def test_rows_beyond_32_bit_offsets():
    """Over 2^31 elements in front of the last row."""
    V, n = 131072, 16400
    x = torch.zeros(n, V, dtype=torch.bfloat16, device="cuda")
    x[-1, 5] = 3.0
    x[-1, V - 1] = 3.0
    values, ids, rest = L().top_logits(x, 3)
    assert ids[-1].tolist() == [5, V - 1, 0] and values[-1].tolist() == [3.0, 3.0, 0.0]
    assert abs(float(rest[-1]) - math.log(V - 3)) < 50 * U + 24 * U
    tokens, _ = L().pick(x, bias_ids=torch.full((n, 1), 9, device="cuda"), bias_values=torch.full((n, 1), 4.0, device="cuda"))
    assert tokens.unique().tolist() == [9]
    y = L().constrain(x, bias_ids=torch.full((n, 1), 9, device="cuda"), bias_values=torch.full((n, 1), 4.0, device="cuda"), out=x)
    assert float(y[-1, 9]) == 4.0 and float(y[-1, V - 1]) == 3.0 and float(y[-2, 5]) == 0.0
    x.requires_grad_(True)
    w = torch.zeros(n, device="cuda")
    w[-1] = 1.0
    loss = L().DistillLoss(denom=1)(x, values, ids, weights=w)
    loss.backward()
    assert float(x.grad[-1].float().abs().max()) > 0 and float(x.grad[:-1].abs().max()) == 0.0


# ---- DistillLoss ---------------------------------------------------------------------------------------------------------
def student(g, n, V, dtype, k, temperature, rest=True, targets=True, weights=True):
    x = rows_like(g, n, V, dtype)
    teacher = x.float() + torch.randn(n, V, generator=g)
    values, ids, tail = ref.top_logits(teacher, k, temperature)
    kw = dict(values=values.float(), ids=ids.clone(), rest=tail.float() if rest else None)
    if targets:
        kw["targets"] = torch.randint(0, V, (n,), generator=g)
        kw["targets"][::3] = ids[::3, 0]                              # a target inside the list
        if n > 4:
            kw["targets"][4] = -100                                   # none
    if weights:
        kw["weights"] = torch.rand(n, generator=g) * 2
        if n > 2:
            kw["weights"][2] = 0.0
    return x, kw


def check_distill(x, kw, temperature, alpha, denom=None, factor=None):
    """Loss and gradient of one call; `factor`: the gradient autograd hands over."""
    leaf = x.cuda().requires_grad_(True)
    loss = L().DistillLoss(temperature, alpha, denom)(leaf, **cuda(kw))
    assert loss.shape == (1,) and loss.dtype == torch.float32
    if factor is None:
        loss.backward()
    else:
        loss.backward(gradient=torch.tensor([factor], device="cuda"))
    within(leaf.grad, loss, x, kw, temperature, alpha, denom, factor)
    return leaf, loss


def within(grad, loss, x, kw, temperature, alpha, denom=None, factor=None):
    """Holds a loss and a gradient against the restatement, with the tolerances that the top of this file derives."""
    wl, wg, rows = ref.distill(x, temperature=temperature, alpha=alpha, denom=denom, **kw)
    d = x.double()
    live = d.isfinite()
    spread = float((d[live].max() - d[live].min())) if bool(live.any()) else 0.0
    az = float(kw["values"].double().nan_to_num(0, 0, 0).abs().max()) / temperature + 40
    w = (kw["weights"] if kw.get("weights") is not None else torch.ones(x.shape[:-1])).double()
    scale = w.sum() / (denom or rows.numel())
    rel = 3 * spread / min(temperature, 1.0) + 100 + 2 * az
    tol = float(scale) * (alpha * temperature ** 2 + 1 - alpha) * rel * U + 4 * U * abs(float(wl))
    assert abs(float(loss.detach()) - float(wl)) <= tol, (float(loss.detach()), float(wl), tol)
    f = 1.0 if factor is None else factor
    got = grad.cpu().double()
    want = wg * f
    n = rows.numel()
    V = x.shape[-1]
    # sizes of the terms of each element: p, the teacher's q, the target
    p = torch.softmax(torch.where(live, d, -math.inf) / temperature, -1) + torch.softmax(torch.where(live, d, -math.inf), -1)
    p = p.nan_to_num(0).reshape(n, V)
    size = p.clone()
    ids = kw["ids"].reshape(n, -1)
    there = (ids >= 0) & (ids < V)
    size.scatter_add_(1, ids.clamp(0, V - 1), there.double())
    if kw.get("rest") is not None:
        size += p * 0 + torch.softmax(torch.where(live, d, -math.inf).reshape(n, V).scatter(1, torch.where(there, ids, 0), -math.inf)
                                      / temperature, -1).nan_to_num(0)
    if kw.get("targets") is not None:
        t = kw["targets"].reshape(n, 1)
        size.scatter_add_(1, t.clamp(0, V - 1), ((t >= 0) & (t < V)).double())
    coef = (w.reshape(n, 1) / (denom or n)) * (alpha * temperature + 1 - alpha) * abs(f)
    bound = (coef * size * rel * U).reshape(x.shape) + HALF[x.dtype] * want.abs() + TINY[x.dtype]
    bad = (got - want).abs() > bound
    assert not bool(bad.any()), (float(((got - want).abs() / bound).max()), bad.nonzero()[0].tolist())


DSHAPES = [(1, 1, 1), (3, 2, 1), (40, 29, 8), (7, 29, 29), (6, 64, 10), (5, 130, 100), (4, 513, 20), (3, 1000, 128), (5, 4099, 64), (6, 8193, 50),
           (5, 32000, 64), (3, 50021, 20), (3, 70001, 64), (2, 131072, 128), (1, 300007, 30), (1, 1048576, 9)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,V,k", DSHAPES)
def test_distill(n, V, k, dtype):
    g = gen(V + k)
    denom = n / 256.0 if dtype == torch.float16 else None     # small gradients vanish in float16 without a loss scale
    for rest, alpha, temperature in ((True, 0.7, 2.0), (False, 1.0, 1.0), (True, 1.0, 1.0), (False, 0.4, 4.0),
                                     (True, 0.5, 3.0), (False, 0.3, 0.7), (True, 1.0, 5.0), (True, 0.0, 2.0), (False, 0.5, 1.0)):
        x, kw = student(g, n, V, dtype, k, temperature, rest, alpha < 1, n % 2 == 1)
        check_distill(x, kw, temperature, alpha, denom)


@pytest.mark.parametrize("V", [29, 700, 9000, 40000, 140000])
def test_distill_of_rows_that_are_not_ordinary(V):
    g = gen(V)
    n, k = 12, 10
    x, kw = student(g, n, V, torch.float32, k, 2.0)
    kw["weights"][:] = 1.0
    kw["weights"][2] = 0.0
    x[2] = math.nan                                # a padded row may hold anything
    kw["values"][2] = math.inf
    kw["ids"][0] = -1                              # nothing in the list: one class on both sides
    kw["ids"][1, 3:] = V + 5                       # padding is no class
    kw["values"][1, 3:] = math.nan                 # ... and its values are not looked at
    kw["ids"][3, 4] = kw["ids"][3, 2]              # the same id twice
    kw["ids"][3, 7] = kw["ids"][3, 2]
    kw["values"][5, 1:] = -math.inf                # teacher: listed, but impossible
    kw["rest"][6] = -math.inf                      # teacher: nothing outside the list
    kw["targets"][7] = V                           # no class
    kw["targets"][8] = kw["ids"][8, k - 1]
    outside = torch.ones(V, dtype=torch.bool)
    outside[kw["ids"][9]] = False
    x[9, outside.nonzero()[1:4, 0]] = -math.inf    # student: tokens that cannot come
    kw["targets"][9] = kw["ids"][9, 0]
    x[10] = torch.finfo(torch.float32).min         # masked with the type's lowest value, but for the list and one more
    x[10, kw["ids"][10]] = torch.randn(k, generator=g)
    x[10, outside.nonzero()[5, 0]] = 0.5
    kw["targets"][10] = kw["ids"][10, 1]
    x[11, kw["ids"][11]] += 200                    # the rest lies far below the list
    keep = [i for i in range(n) if i != 10]
    pick = lambda d, at: {a: (b[at] if torch.is_tensor(b) else b) for a, b in d.items()}  # noqa: E731
    check_distill(x[keep], pick(kw, keep), 2.0, 0.6)
    check_distill(x[keep], dict(pick(kw, keep), rest=None), 2.0, 0.6)
    for temperature in (1.0, 3.0, 4.0):   # (the lists are numbers like any others at these temperatures)
        check_distill(x[keep], pick(kw, keep), temperature, 0.6)
    # the row of lowest values by itself: its spread is the type's, the bound above would say nothing
    leaf = x[10:11].cuda().requires_grad_(True)
    one = cuda(pick(kw, [10]))
    loss = L().DistillLoss(2.0, 0.6)(leaf, **one)
    loss.backward()
    y = x[10:11].clone()
    y[y < -1e30] = -1e4
    wl, wg, _ = ref.distill(y, temperature=2.0, alpha=0.6, **pick(kw, [10]))
    assert abs(float(loss.detach()) - float(wl)) <= 300 * U * (1 + abs(float(wl)))
    assert float((leaf.grad.cpu().double() - wg).abs().max()) <= 300 * U


@pytest.mark.parametrize("V", [29, 700, 9000, 40000, 140000])
def test_distill_of_a_teacher_that_is_no_distribution(V):
    """NaN or +inf among the entries or in the rest: the loss says so, and every other row's gradient is as ever."""
    g = gen(V)
    n, k = 4, 6
    x, kw = student(g, n, V, torch.float32, k, 2.0, weights=False)
    clean = x.cuda().requires_grad_(True)
    L().DistillLoss(2.0, 0.6)(clean, **cuda(kw)).backward()
    for bad in (math.nan, math.inf):
        for where in ("values", "rest", "only entry", "without a rest"):
            mine = {a: t.clone() for a, t in kw.items()}
            if where == "rest":
                mine["rest"][1] = bad
            else:
                mine["values"][1, 3] = bad
            if where == "only entry":
                mine["ids"][1, :3] = mine["ids"][1, 4:] = -1
                mine["rest"][1] = -math.inf
            if where == "without a rest":
                mine["rest"] = None
                mine["ids"][1, :3] = mine["ids"][1, 4:] = -1
            leaf = x.cuda().requires_grad_(True)
            loss = L().DistillLoss(2.0, 0.6)(leaf, **cuda(mine))
            loss.backward()
            assert bool(loss.detach().isnan()), (bad, where)
            assert bool(leaf.grad[1, mine["ids"][1, 3].item()].isnan()), (bad, where)
            if where != "without a rest":
                assert torch.equal(leaf.grad[[0, 2, 3]], clean.grad[[0, 2, 3]]), (bad, where)
            w = torch.ones(n)
            w[1] = 0.0
            assert bool(L().DistillLoss(2.0, 0.6)(leaf.detach(), weights=w.cuda(), **cuda(mine)).isfinite())
            assert bool(L().DistillLoss(2.0, 0.0)(leaf.detach(), **cuda(mine)).isfinite())


def test_distill_rows_without_anything():
    """No entry, no rest, no target: no loss and a gradient of exactly zero."""
    x = torch.randn(4, 50, generator=gen(1)).cuda().requires_grad_(True)
    ids = torch.full((4, 3), -1).cuda()
    values = torch.full((4, 3), math.nan).cuda()
    loss = L().DistillLoss(2.0, 0.5)(x, values, ids, targets=torch.full((4,), -100).cuda())
    loss.backward()
    assert float(loss.detach()) == 0.0 and float(x.grad.abs().max()) == 0.0
    empty = torch.zeros(0, 50).cuda().requires_grad_(True)
    loss = L().DistillLoss()(empty, values[:0], ids[:0])
    loss.backward()
    assert float(loss.detach()) == 0.0 and empty.grad.shape == (0, 50)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [29, 9001])
def test_distill_on_views(V, dtype):
    """Time-major logits handed over batch-first: the gradient has their layout; rows with gaps and shared rows work too."""
    g = gen(V)
    T, B, k = 5, 3, 6
    x, kw = student(g, T * B, V, dtype, k, 2.0)
    base = x.view(T, B, V)
    kw = {a: b.view(B, T, *b.shape[1:]) for a, b in kw.items()}
    denom = 15 / 64.0
    leaf = base.cuda().requires_grad_(True)
    loss = L().DistillLoss(2.0, 0.5, denom)(leaf.transpose(0, 1), **cuda(kw))
    loss.backward()
    # (sums run in another order where rows start at other offsets from a 16-byte boundary: every layout is held to the
    # restatement by the tolerances at the top of this file, not to another layout's bits)
    packed = base.transpose(0, 1).contiguous()
    within(leaf.grad.transpose(0, 1), loss, packed, kw, 2.0, 0.5, denom)
    check_distill(packed, kw, 2.0, 0.5, denom)
    wide = torch.zeros(B, T, V + 5, dtype=dtype)
    wide[..., 2:V + 2] = packed
    wide = wide.cuda().requires_grad_(True)
    loss = L().DistillLoss(2.0, 0.5, denom)(wide[..., 2:V + 2], **cuda(kw))
    loss.backward()
    within(wide.grad[..., 2:V + 2], loss, packed, kw, 2.0, 0.5, denom)
    assert float(wide.grad[..., :2].abs().max()) == 0.0 == float(wide.grad[..., V + 2:].abs().max())
    one = base[:1, 0].cuda().requires_grad_(True)     # one row for every entry of the list: gradients of a broadcast input add up
    row_kw = {a: b.reshape(B * T, *b.shape[2:]) for a, b in cuda(kw).items()}
    L().DistillLoss(2.0, 0.5, denom)(one.expand(B * T, V), **row_kw).backward()
    many = base[:1, 0].repeat(B * T, 1).cuda().requires_grad_(True)
    L().DistillLoss(2.0, 0.5, denom)(many, **row_kw).backward()
    want = many.grad.double().sum(0)
    assert float((one.grad[0].double() - want).abs().max()) <= B * T * HALF[dtype] * float(many.grad.double().abs().sum(0).max())


def test_distill_factors_and_second_walks():
    from speech_amd import ops
    g = gen(9)
    x, kw = student(g, 6, 3001, torch.bfloat16, 12, 2.0)
    check_distill(x, kw, 2.0, 0.5, factor=-3.25)
    check_distill(x, kw, 2.0, 0.5, factor=0.0)
    dev = cuda(kw)
    leaf = x.cuda().requires_grad_(True)
    loss = L().DistillLoss(2.0, 0.5)(leaf, **dev)
    ops.backward(loss)
    first = leaf.grad
    leaf.grad = None
    other = L().DistillLoss(2.0, 0.5)(leaf, **dev)
    other.backward(retain_graph=True)                      # autograd's own seed
    assert torch.equal(leaf.grad, first)
    kept, leaf.grad = leaf.grad, None
    kept.zero_()                                           # what a caller does to a gradient reaches no later walk
    other.backward(retain_graph=True)
    assert torch.equal(leaf.grad, first)
    leaf.grad = None
    other.backward(gradient=torch.tensor([0.5], device="cuda"))
    check, _ = check_distill(x, kw, 2.0, 0.5, factor=0.5)
    assert torch.equal(leaf.grad, check.grad)
    # gradients add up over two losses of the same leaf, and the loss is a number like any other
    leaf.grad = None
    (2 * L().DistillLoss(2.0, 0.5)(leaf, **dev) + L().DistillLoss(1.0)(leaf, dev["values"], dev["ids"])).backward()
    a, _ = check_distill(x, kw, 2.0, 0.5, factor=2.0)
    b, _ = check_distill(x, {"values": kw["values"], "ids": kw["ids"]}, 1.0, 1.0)
    assert torch.equal(leaf.grad, a.grad + b.grad)
    with torch.no_grad():
        assert not L().DistillLoss(2.0, 0.5)(leaf, **dev).requires_grad
    # changed in place between the passes: a walk that needs the logits again says so; a second derivative is refused
    from speech_amd._lib import SpeechAmdError
    loss = L().DistillLoss(2.0, 0.5)(leaf, **dev)
    with torch.no_grad():
        leaf += 1
    with pytest.raises(RuntimeError, match="in ?place"):
        loss.backward()
    with pytest.raises(SpeechAmdError, match="once"):
        torch.autograd.grad(L().DistillLoss(2.0, 0.5)(leaf, **dev), leaf, create_graph=True)
    for name in ("values", "ids", "rest", "targets", "weights"):
        mine = {a: v.clone() for a, v in dev.items()}
        loss = L().DistillLoss(2.0, 0.5)(leaf, **mine)
        mine[name].zero_()
        with pytest.raises(RuntimeError, match="in place"):
            (2 * loss).backward()
    # the walk frees the logits, and says so to a second one
    loss = L().DistillLoss(2.0, 0.5)(leaf, **dev)
    (2 * loss).backward()
    with pytest.raises(RuntimeError, match="second time"):
        (2 * loss).backward()
    # what a teacher made in inference mode is as good as any other
    with torch.inference_mode():
        given = {a: v.clone() for a, v in dev.items()}
        L().constrain(leaf, bias_ids=dev["ids"], bias_values=dev["values"])
    leaf.grad = None
    (2 * L().DistillLoss(2.0, 0.5)(leaf, **given)).backward()
    by_lists, leaf.grad = leaf.grad, None
    (2 * L().DistillLoss(2.0, 0.5)(leaf, **dev)).backward()
    assert torch.equal(by_lists, leaf.grad)


def test_distill_gradient_against_differences():
    """Along a direction: the loss is read from the kernel, in steps that its float32 noise does not drown."""
    g = gen(4)
    x, kw = student(g, 8, 500, torch.float32, 16, 2.0)
    leaf, _ = check_distill(x, kw, 2.0, 0.5)
    u = torch.randn(x.shape, generator=g)
    h = 2.0 ** -5
    loss = L().DistillLoss(2.0, 0.5)
    at = [float(loss((x + s * h * u).cuda(), **cuda(kw))) for s in (-2, -1, 1, 2)]
    slope = (8 * (at[2] - at[1]) - (at[3] - at[0])) / (12 * h)
    want = float((leaf.grad.cpu().double() * u.double()).sum())
    # fourth-order differences: h^4 / 30 times the fifth derivative (below 100 here), and 1.5 / h times the noise of a loss near 3
    assert abs(slope - want) < 100 * h ** 4 / 30 + 1.5 / h * 300 * U * 3


def test_distill_refuses():
    from speech_amd._lib import SpeechAmdError
    x, kw = student(gen(2), 4, 30, torch.float32, 5, 1.0)
    kw = cuda(kw)
    x = x.cuda()
    for bad in (dict(values=kw["values"].double()), dict(values=kw["values"][:3]), dict(ids=kw["ids"].int()), dict(ids=kw["ids"][:, :4]),
                dict(rest=kw["rest"][:, None]), dict(targets=kw["targets"].int()), dict(weights=kw["weights"].cpu()),
                dict(ids=kw["ids"].t().contiguous().t())):
        with pytest.raises(SpeechAmdError):
            L().DistillLoss(1.0, 0.5)(x, **dict(kw, **bad))
    with pytest.raises(SpeechAmdError):
        L().DistillLoss()(x.double(), kw["values"], kw["ids"])
    with pytest.raises(SpeechAmdError):
        L().top_logits(x, 31)


# ---- streams, graphs, the operators together --------------------------------------------------------------------------------
def test_on_another_stream_and_twice_at_once():
    g = gen(6)
    x = rows_like(g, 40, 20011, torch.float32)
    kw = constraints(g, 40, 20011, 100, 8, True)
    want = [L().pick(x.cuda(), **cuda(kw)), L().top_logits(x.cuda(), 30)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            dev, k2 = x.cuda(), cuda(kw)
            for _ in range(3):
                got.append((L().pick(dev, **k2), L().top_logits(dev, 30)))
    torch.cuda.synchronize()
    for p, t in got:
        assert all(torch.equal(a, b) for a, b in zip(p, want[0])) and all(torch.equal(a, b) for a, b in zip(t, want[1]))


def test_captured_graphs():
    """Two graphs captured next to each other and an eager program between their replays: each replay is the eager result."""
    g = gen(8)
    n, V = 24, 20011
    inputs = [rows_like(g, n, V, torch.bfloat16).cuda() for _ in range(4)]
    kw = cuda(constraints(g, n, V, 64, 8, True))
    _, sk = student(g, n, V, torch.bfloat16, 16, 2.0)
    sk = cuda(sk)
    static = [inputs[0].clone().requires_grad_(True), inputs[1].clone().requires_grad_(True)]

    def everything(x):
        x.grad = None
        loss = L().DistillLoss(2.0, 0.5)(x, **sk)
        loss.backward()
        y = x.detach()
        return [loss.detach(), x.grad, *L().pick(y, **kw), L().constrain(y, **kw), *L().top_logits(y, 20, 2.0)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in static:
            everything(x)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x in static:
        graph = torch.cuda.CUDAGraph()
        x.grad = None
        with torch.cuda.graph(graph):
            outs.append(everything(x))
        graphs.append(graph)
    for trip in range(4):
        for i in (0, 1):
            with torch.no_grad():
                static[i].copy_(inputs[(trip + i) % 4])
        graphs[0].replay()
        graphs[1].replay()
        want = [everything(inputs[(trip + i) % 4].clone().requires_grad_(True)) for i in (0, 1)]
        torch.cuda.synchronize()
        for i in (0, 1):
            for a, b in zip(outs[i], want[i]):
                assert torch.equal(a.float().nan_to_num(nan=1e30), b.float().nan_to_num(nan=1e30)), (trip, i)


@pytest.mark.parametrize("V,dtype", [(140000, torch.float32), (300007, torch.float32), (280001, torch.bfloat16)])
def test_captured_graphs_of_rows_beyond_the_registers(V, dtype):
    """Rows that the loss keeps in LDS, more than 48 KB of it: the kernel's limit is raised inside the capture too."""
    g = gen(V)
    n = 3
    inputs = [rows_like(g, n, V, dtype).cuda() for _ in range(3)]
    _, sk = student(g, n, V, dtype, 16, 2.0)
    sk = cuda(sk)
    static = inputs[0].clone().requires_grad_(True)

    def step(x):
        x.grad = None
        loss = L().DistillLoss(2.0, 0.5, denom=n / 256.0)(x, **sk)
        loss.backward()
        return [loss.detach(), x.grad]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    static.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for trip in range(4):
        with torch.no_grad():
            static.copy_(inputs[trip % 3])
        graph.replay()
        want = step(inputs[trip % 3].clone().requires_grad_(True))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), trip


def test_same_bits_on_every_run():
    g = gen(12)
    x = rows_like(g, 16, 70001, torch.float32).cuda()
    kw = cuda(constraints(g, 16, 70001, 500, 40, True))
    _, sk = student(g, 16, 70001, torch.float32, 40, 2.0)
    sk["ids"][:, 7] = sk["ids"][:, 3]
    sk = cuda(sk)

    def all_of_it():
        leaf = x.clone().requires_grad_(True)
        loss = L().DistillLoss(2.0, 0.5)(leaf, **sk)
        loss.backward()
        return [loss.detach(), leaf.grad, L().constrain(x, **kw), *L().pick(x, **kw), *L().top_logits(x, 40)]

    want = all_of_it()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(all_of_it(), want))


def test_teacher_to_student_to_answer():
    """The operators as they are used together: a teacher's rows -> its top logits -> a student trained on them -> tokens under a
    grammar that the teacher's choice obeys."""
    g = gen(20)
    n, V, k = 64, 777, 12
    teacher = rows_like(g, n, V, torch.float32).cuda()
    values, ids, rest = L().top_logits(teacher, k, 2.0)
    leaf = torch.zeros(n, V, device="cuda", requires_grad=True)
    loss_fn = L().DistillLoss(2.0)
    first = None
    for _ in range(60):
        leaf.grad = None
        loss = loss_fn(leaf, values, ids, rest=rest)
        loss.backward()
        with torch.no_grad():
            leaf -= 40.0 * leaf.grad
        first = first if first is not None else float(loss.detach())
    assert first > 0 and leaf.grad.isfinite().all()
    allowed = torch.zeros(n, V, dtype=torch.bool)
    allowed.scatter_(1, ids[:, :2].cpu(), True)
    tokens, logp = L().pick(leaf.detach(), mask=L().pack_mask(allowed).cuda())
    assert bool(((tokens == ids[:, 0]) | (tokens == ids[:, 1])).all()) and bool((logp <= 0).all())
    # the answers so far are not to come again: with a heavy penalty the other allowed token is taken
    again, _ = L().pick(leaf.detach(), history=tokens[:, None].contiguous(), presence=1e4, mask=L().pack_mask(allowed).cuda())
    assert bool((again != tokens).all()) and bool(((again == ids[:, 0]) | (again == ids[:, 1])).all())
