"""Refusals of rl_specdec_verify_draft / rl_specdec_verify_tree and of their
Python forms, and known answers of the 64-bit restatement. No GPU: a block of
zeros stands for a handle, since every refusal comes before any device work."""
import ctypes

import numpy as np
import pytest

import rlsampler
import verify as ref

torch = pytest.importorskip("torch")
P = None
X = ctypes.c_void_p(64)  # an address that no refused call looks at


def handle():
    return ctypes.create_string_buffer(4096)


def side(**kw):
    d = dict(logits=64, dtype=0, rows=100, ld=10, temperature=None, mask=None, mask_stride=0, cut=None, cut_stride=0,
             first_row=None)
    d.update(kw)
    return rlsampler._DistRows(**d)


def chain(h, B=2, V=10, K=3, t=None, d=None, drafts=X, n=X, u=X, du=X, acc=X, tok=X):
    return rlsampler.lib().rl_specdec_verify_draft(h, B, V, K, t if t is not None else side(), d, drafts, n, u, du, acc, tok, P, P, P)


def tree(h, B=2, V=10, N=4, t=None, d=None, tokens=X, parent=X, n=X, u=X, du=X, acc=X, tok=X):
    return rlsampler.lib().rl_specdec_verify_tree(h, B, V, N, t if t is not None else side(), d, tokens, parent, n, u, du, acc, P, tok, P, P, P)


@pytest.mark.parametrize("call", [chain, tree])
def test_refusals(call):
    h = handle()
    assert call(None) == rlsampler.RL_ERR_INVALID_ARG and "handle" in rlsampler.last_error()
    assert call(h, B=0) == rlsampler.RL_OK
    for bad in (dict(B=-1), dict(V=0), dict(n=P), dict(u=P), dict(du=P), dict(acc=P), dict(tok=P), dict(t=side(logits=None)),
                dict(t=side(dtype=7)), dict(t=side(ld=9)), dict(t=side(rows=-1)), dict(t=side(logits=66)),
                dict(t=side(mask=64, mask_stride=0)), dict(t=side(cut=64, cut_stride=-1)), dict(d=side(ld=3)),
                dict(d=side(logits=65, dtype=1))):
        assert call(h, **bad) == rlsampler.RL_ERR_INVALID_ARG, bad
        assert rlsampler.last_error(), bad
    for bad in (dict(t=side(rows=7)), dict(d=side(rows=5)), dict(V=(1 << 30) + 1)):
        assert call(h, **bad) == rlsampler.RL_ERR_SHAPE, bad


def test_refusals_of_one_form():
    h = handle()
    assert chain(h, K=-1) == rlsampler.RL_ERR_INVALID_ARG
    assert chain(h, K=256) == rlsampler.RL_ERR_SHAPE
    assert chain(h, drafts=P) == rlsampler.RL_ERR_INVALID_ARG
    assert tree(h, N=0) == rlsampler.RL_ERR_INVALID_ARG
    assert tree(h, N=257) == rlsampler.RL_ERR_SHAPE
    assert tree(h, tokens=P) == rlsampler.RL_ERR_INVALID_ARG
    assert tree(h, parent=P) == rlsampler.RL_ERR_INVALID_ARG


def test_python_forms_refuse():
    x = torch.zeros(8, 40)
    i = torch.zeros(2, 3, dtype=torch.int32)
    for bad in (dict(logits=x[0]), dict(logits=x.t()), dict(logits=x.double()), dict(logits=x, temperature=torch.zeros(2, dtype=torch.float64)),
                dict(logits=x, mask=torch.zeros(8, 2)), dict(logits=x, mask=torch.zeros(7, 2, dtype=torch.int32)),
                dict(logits=x, cut=torch.zeros(7, dtype=torch.int32)), dict(logits=x, temperature=torch.zeros(4)[::2])):
        with pytest.raises(ValueError):
            rlsampler.DistRows(**bad)
    s = rlsampler.Sampler.__new__(rlsampler.Sampler)
    s.h = None
    t = rlsampler.DistRows(x)
    u, n, du = torch.zeros(2, 3), torch.zeros(2, dtype=torch.int32), torch.zeros(2)
    good = (i, n, u, du)
    for k, wrong in enumerate((i.long(), torch.zeros(3, dtype=torch.int32), torch.zeros(2, 4), torch.zeros(2, dtype=torch.float64))):
        args = list(good)
        args[k] = wrong
        with pytest.raises(ValueError):
            s.specdec_verify_draft(t, *args)
    with pytest.raises(ValueError):
        s.specdec_verify_draft(t, *good, draft=rlsampler.DistRows(torch.zeros(6, 41)))
    with pytest.raises(ValueError):
        s.specdec_verify_tree(t, i, i.t().contiguous().t(), n, u, du)
    with pytest.raises(ValueError):
        s.specdec_verify_draft(rlsampler.DistRows(x, mask=torch.zeros(8, 1, dtype=torch.int32)), *good)
    with pytest.raises(ValueError):
        s.specdec_verify_draft(rlsampler.DistRows(x, temperature=torch.zeros(3)), *good)


def test_restatement_known_answers():
    p, q = np.log([0.5, 0.3, 0.2]), np.log([0.2, 0.3, 0.5])
    one = lambda u, du, x, q_=q: ref.walk(lambda i: ref.dist(p), lambda i: None if q_ is None else ref.dist(q_), lambda i: [1] if i == 0 else [], lambda c: x, lambda c: u, du)  # noqa: E731
    assert one(0.99, 0.1, 0).tokens == [0, 0]  # p > q: always accepted, then from p
    r = one(0.5, 0.9, 2)  # 0.5 * 0.5 >= 0.2: refused, the residual is id 0 alone
    assert r.path == [] and r.tokens == [0]
    assert one(0.3, 0.6, 2).tokens == [2, 1]
    r = one(0.6, 0.5, 0, None)  # given: accepted with p = 0.5
    assert r.path == [] and r.tokens == [1]
    assert ref.dist([0.0, np.nan]) is None and ref.dist([-np.inf, -np.inf]) is None
    assert ref.dist([1.0, 1.0, 0.0], 0.0).tolist() == [1.0, 0.0, 0.0]
    m = np.array([0b010], np.uint32)
    assert ref.dist([np.nan, 1.0, np.inf], 1.0, m).tolist() == [0.0, 1.0, 0.0]
    assert ref.dist([1.0, 2.0, 1.0], 1.0, None, 0)[2] == 0.0
    # siblings: w after two refusals is max(p - C q, 0) with C = 1 + S
    q2 = np.log([0.1, 0.6, 0.3])
    w = ref.walk(lambda i: ref.dist(p), lambda i: ref.dist(q2), lambda i: [1, 2] if i == 0 else [], lambda c: 1, lambda c: 1.0, 0.5).w
    s1 = 0.4
    np.testing.assert_allclose(w, np.maximum(np.array([0.5, 0.3, 0.2]) - (1 + s1) * np.array([0.1, 0.6, 0.3]), 0), atol=1e-12)
