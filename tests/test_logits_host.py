"""speech_amd.logits without a GPU: what it refuses (before anything is launched), pack_mask, and the restatement's own gradient
against differences."""
import ctypes
import math

import pytest
import torch

from oracle import logits_ref
from speech_amd import _lib, logits as L
from speech_amd._lib import SpeechAmdError


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 8)
    for call in (lambda: L.constrain(x), lambda: L.pick(x), lambda: L.top_logits(x, 2),
                 lambda: L.DistillLoss()(x, torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int64))):
        with pytest.raises(SpeechAmdError, match="GPU"):
            call()


@pytest.mark.parametrize("x", [torch.zeros(8), torch.zeros(2, 8, dtype=torch.float64), torch.zeros(2, 8, dtype=torch.int64),
                               torch.zeros(8, 2).t(), torch.zeros(2, 0), torch.zeros(1, 1).expand(2, L.VOCAB_MAX + 1), "logits"])
def test_logits_of_another_form_are_refused(x):
    for call in (lambda: L.constrain(x), lambda: L.pick(x), lambda: L.top_logits(x, 1)):
        with pytest.raises(SpeechAmdError):
            call()


def _check(rows=3, V=40, **kw):
    full = dict(history=None, lengths=None, repetition=None, presence=None, frequency=None, bias_ids=None, bias_values=None,
                mask=None, states=None)
    full.update(kw)
    return L._constraints(rows, V, torch.device("cpu"), *full.values())


H = torch.zeros(3, 5, dtype=torch.int64)
I32 = torch.zeros(3, dtype=torch.int32)


@pytest.mark.parametrize("kw", [
    dict(history=H.int()), dict(history=H[:2]), dict(history=H[0]), dict(history=H.t()[:3].t()[:, ::2]),
    dict(history=torch.zeros(1, 1, dtype=torch.int64).expand(3, L.LIST_MAX + 1)),
    dict(lengths=I32), dict(history=H, lengths=I32.long()), dict(history=H, lengths=I32[:2]), dict(history=H, lengths=[1, 2, 3]),
    dict(repetition=1.2), dict(history=H, repetition=0.0), dict(history=H, repetition=-1.0), dict(history=H, repetition=math.inf),
    dict(history=H, presence=math.nan), dict(history=H, frequency=torch.zeros(2)), dict(history=H, frequency=torch.zeros(3).double()),
    dict(bias_ids=H), dict(bias_values=torch.zeros(3, 5)), dict(bias_ids=H, bias_values=torch.zeros(3, 4)),
    dict(bias_ids=H, bias_values=torch.zeros(3, 5).half()), dict(bias_ids=H, bias_values=torch.zeros(3, 10)[:, :5]),
    dict(mask=torch.zeros(3, 1, dtype=torch.int32)), dict(mask=torch.zeros(3, 2)), dict(mask=torch.zeros(2, 2, dtype=torch.int32)),
    dict(mask=torch.zeros(0, 2, dtype=torch.int32), states=I32), dict(states=I32),
    dict(mask=torch.zeros(2, 2, dtype=torch.int32), states=I32.long()), dict(mask=torch.zeros(1, 2, dtype=torch.int32).expand(4, 2), states=I32),
])
def test_constraints_of_another_form_are_refused(kw):
    with pytest.raises(SpeechAmdError):
        _check(**kw)


def test_constraints_as_the_library_reads_them():
    ids, values = torch.zeros(3, 4, dtype=torch.int64), torch.zeros(3, 4)
    wide = torch.zeros(3, 9, dtype=torch.int64)[:, :5]
    c = _check(history=wide, lengths=I32, repetition=1.5, presence=torch.zeros(3), bias_ids=ids, bias_values=values,
               mask=torch.zeros(7, 3, dtype=torch.int32), states=I32)
    assert (c.history, c.history_ld, c.history_len) == (wide.data_ptr(), 9, 5)
    assert c.repetition is None and c.repetition_all == 1.5 and c.presence and c.frequency_all == 0.0
    assert (c.n_bias, c.bias_ld, c.n_states, c.mask_ld) == (4, 4, 7, 3)


@pytest.mark.parametrize("k", [0, -1, 9, 129])
def test_k_out_of_range_is_refused(k):
    class Fake(torch.Tensor):  # a CPU tensor that says it is on the GPU: every check runs, nothing is launched
        is_cuda = True

    with pytest.raises(SpeechAmdError, match="k must be"):
        L.top_logits(torch.zeros(2, 8).as_subclass(Fake), k)


def test_parameters_of_the_loss_are_checked():
    for kw in (dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.inf), dict(alpha=1.1), dict(alpha=-0.1),
               dict(alpha=math.nan), dict(denom=0.0), dict(denom=-2), dict(denom=math.nan)):
        with pytest.raises(SpeechAmdError):
            L.DistillLoss(**kw)
    x, v, i = torch.zeros(2, 8), torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int64)
    with pytest.raises(SpeechAmdError, match="targets"):
        L.DistillLoss(alpha=0.5)(x, v, i)
    with pytest.raises(SpeechAmdError, match="k"):
        L.DistillLoss()(x, torch.zeros(2, 129), torch.zeros(2, 129, dtype=torch.int64))
    for t in (0.0, -1.0, math.nan, math.inf, 1e-9, 1e9):
        with pytest.raises(SpeechAmdError, match="temperature"):
            L._temperature(t)


def test_numbers_in_place_of_rows_are_refused():
    x, v, i = torch.zeros(2, 8), torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int64)
    for logits, values in ((x, v[0, 0]), (x[0, 0], v), (x, 1.0), (1.0, v), (x, None)):
        with pytest.raises(SpeechAmdError):
            L.DistillLoss()(logits, values, i)
    for call in (L.constrain, L.pick, lambda t: L.top_logits(t, 1)):
        with pytest.raises(SpeechAmdError):
            call(x[0, 0])


def test_the_c_entries_refuse_before_they_launch():
    lib = _lib.lib()
    c = _lib.saConstraints()
    c.repetition_all = 1.0
    bad = 2  # CTC_STATUS_INVALID_VALUE
    P = 1 << 12  # never dereferenced: every call below is refused on its sizes, or has no rows
    ref = ctypes.byref(c)
    assert lib.sa_logits_constrain(P, 8, 3, P, 8, 1, 8, ref, None) == bad                    # type
    assert lib.sa_logits_constrain(P, 8, 0, P, 8, 1, 0, ref, None) == bad                    # V
    assert lib.sa_logits_constrain(P, 8, 0, P, 8, 1, L.VOCAB_MAX + 1, ref, None) == bad
    assert lib.sa_logits_constrain(P, 8, 0, P, 8, -1, 8, ref, None) == bad
    assert lib.sa_logits_constrain(P, 8, 0, P, 8, 1, 8, None, None) == bad
    assert lib.sa_logits_constrain(None, 8, 0, P, 8, 1, 8, ref, None) == bad
    assert lib.sa_logits_constrain(None, 8, 0, None, 8, 0, 8, ref, None) == 0                # no rows: nothing to do
    assert lib.sa_logits_pick(P, 8, 0, 1, 8, ref, None, P, None, 0, None) == bad
    assert lib.sa_logits_pick(P, 8, 0, 1, 200000, ref, P, P, None, 0, None) == bad           # needs a workspace
    c.history_len = 4
    assert lib.sa_logits_pick(P, 8, 0, 1, 8, ref, P, P, None, 0, None) == bad                # a history without one
    c.history_len = L.LIST_MAX + 1
    c.history = P
    assert lib.sa_logits_pick(P, 8, 0, 1, 8, ref, P, P, None, 0, None) == bad
    c.history_len, c.mask, c.n_states, c.mask_ld = 0, P, 1, 0
    assert lib.sa_logits_pick(P, 8, 0, 1, 8, ref, P, P, None, 0, None) == bad                # mask rows too short
    c.mask_ld = 1
    assert lib.sa_logits_pick(P, 8, 0, 2, 8, ref, P, P, None, 0, None) == bad                # two requests, one row, no states

    def top(x=P, dtype=0, rows=1, V=8, k=2, t=1.0, n_inner=1):
        return lib.sa_top_logits(x, V, 0, n_inner, dtype, rows, V, k, t, P, P, P, None, 0, None)
    assert top(k=0) == top(k=9) == top(V=500, k=129) == top(t=0.0) == top(t=math.inf) == top(t=math.nan) == bad
    assert top(x=None) == top(dtype=-1) == top(rows=-1) == top(n_inner=0) == bad and top(x=None, rows=0) == 0
    assert lib.sa_top_logits_workspace_bytes(0, 8, 2, 0) == 0

    def dis(x=P, dx=P, V=8, k=2, t=1.0, alpha=1.0, rows=1, loss=P, loss_rows=P):
        return lib.sa_distill_loss(x, dx, V, 0, 1, 0, rows, V, P, P, None, k, None, None, t, alpha, 1.0, None, 0, loss_rows,
                                   loss, None)
    assert dis(k=0) == dis(k=129) == dis(t=0.0) == dis(t=math.nan) == dis(alpha=1.5) == dis(alpha=math.nan) == bad
    assert top(t=1e-9) == top(t=1e9) == dis(t=1e-9) == dis(t=1e9) == bad
    assert dis(x=None) == dis(rows=-1) == dis(loss_rows=None) == dis(loss=None, dx=None) == dis(V=0) == bad
    # more rows than a launch has threads for
    assert top(rows=1 << 28) == top(rows=1 << 27, V=100) == top(rows=1 << 26, V=500) == top(rows=1 << 40) == bad
    assert dis(rows=1 << 26) == dis(rows=1 << 24, V=5000) == dis(rows=1 << 40) == bad
    assert lib.sa_top_logits_workspace_bytes(1 << 40, 8, 2, 0) == 0
    c = _lib.saConstraints()
    ref = ctypes.byref(c)
    assert lib.sa_logits_pick(P, 8, 0, 1 << 24, 8, ref, P, P, None, 0, None) == bad
    assert lib.sa_logits_constrain(P, 8, 0, P, 8, 1 << 24, 8, ref, None) == bad


def test_a_batch_without_requests_is_no_error():
    """Empty tensors have no address: with no row there is nothing to read, whatever lists and masks come along."""
    none = torch.zeros(0, 5, dtype=torch.int64)
    i32 = torch.zeros(0, dtype=torch.int32)
    words = L.pack_mask(torch.zeros(0, 40, dtype=torch.bool))
    assert words.shape == (0, 2) and words.dtype == torch.int32
    lib = _lib.lib()
    for kw in (dict(history=none), dict(history=none, lengths=i32, repetition=torch.zeros(0), presence=0.5),
               dict(bias_ids=none, bias_values=torch.zeros(0, 5)), dict(mask=words), dict(mask=words, states=i32),
               dict(mask=torch.zeros(3, 2, dtype=torch.int32), states=i32)):
        c = ctypes.byref(_check(rows=0, **kw))
        assert lib.sa_logits_constrain(None, 40, 0, None, 40, 0, 40, c, None) == 0, list(kw)
        assert lib.sa_logits_pick(None, 40, 0, 0, 40, c, None, None, None, 0, None) == 0, list(kw)


def test_the_constrained_decode_refuses_before_it_launches():
    lib = _lib.lib()
    P, bad = 1 << 12, 2
    plist = (ctypes.c_void_p * 11)(*[P] * 11)
    c = _lib.saConstraints()
    c.repetition_all = 1.0

    def run(con=c, end=3, max_len=4, states=None, following=None, ws=1 << 30, B=2, K=13):
        return lib.sa_s2s_greedy_decode_constrained(P, plist, B, 20, 16, 16, 15, K, 1.0, end, max_len, 8,
                                                    None if con is None else ctypes.byref(con), 1, states, following, P, P, P, ws,
                                                    None)
    assert run(con=None) == run(end=-1) == run(end=13) == run(max_len=0) == run(max_len=L.LIST_MAX) == bad
    assert run(following=P) == run(ws=16) == run(B=0) == bad
    c.mask, c.n_states, c.mask_ld = P, 2, 1
    assert run(states=None) == bad


def test_what_out_may_share_with_the_logits():
    b = torch.zeros(6, 10)

    def meet(x, y):
        return L._overlap(x, x.stride(0), y, y.stride(0), x.shape[0], x.shape[1])
    assert not meet(b, b) and not meet(b, b.clone()) and not meet(b[:3], b[3:]) and not meet(b[3:], b[:3])
    assert not meet(b[:, :5], b[:, 5:]) and not meet(b[:, 5:], b[:, :5]) and not meet(b[::2], b[1::2])
    assert not meet(b[:, :4], b[:, 6:]) and not meet(b[:1], b[:1]) and not meet(b[:0], b[:0])
    assert meet(b[:4], b[1:5]) and meet(b[1:5], b[:4]) and meet(b[:, :6], b[:, 4:]) and meet(b[:, 4:], b[:, :6])
    assert meet(b[:2, :5], b[::2][:2, :5]) and meet(b[:1].expand(3, 10), b[:3]) and meet(b.view(1, 60)[:, :20], b.view(1, 60)[:, 10:30])
    assert meet(b[:3, :8], b.as_strided((3, 8), (10, 1), 13))


def test_pack_mask():
    g = torch.Generator().manual_seed(3)
    for V in (1, 31, 32, 33, 64, 100):
        allowed = torch.rand(5, V, generator=g) < 0.5
        words = L.pack_mask(allowed)
        assert words.dtype == torch.int32 and words.shape == (5, (V + 31) // 32)
        x = logits_ref.constrain(torch.zeros(5, V), mask=words)
        assert torch.equal(x == 0, allowed)
    for bad in (torch.ones(3, 4), torch.ones(4, dtype=torch.bool), torch.ones(3, 0, dtype=torch.bool)):
        with pytest.raises(SpeechAmdError):
            L.pack_mask(bad)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("alpha", [0.0, 0.6, 1.0])
def test_restatement_gradient_against_differences(rest, alpha):
    g = torch.Generator().manual_seed(1)
    n, V, k = 3, 11, 4
    x = torch.randn(n, V, generator=g, dtype=torch.float64)
    values, ids, tail = logits_ref.top_logits(x + torch.randn(n, V, generator=g), k, 2.0)
    ids = ids.clone()
    ids[1, 2] = -1           # absent
    ids[2, 1] = ids[2, 0]    # the same id twice
    kw = dict(rest=tail if rest else None, targets=torch.tensor([3, -100, 10]), weights=torch.tensor([1.0, 0.5, 2.0]),
              temperature=2.0, alpha=alpha)
    _, grad, _ = logits_ref.distill(x, values, ids, **kw)
    h = 1e-6
    for i in range(n):
        for v in range(V):
            up, down = x.clone(), x.clone()
            up[i, v] += h
            down[i, v] -= h
            d = (logits_ref.distill(up, values, ids, **kw)[0] - logits_ref.distill(down, values, ids, **kw)[0]) / (2 * h)
            assert abs(float(d - grad[i, v])) < 1e-8
