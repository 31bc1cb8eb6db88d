"""Refusals of rl_lmhead_q4_* and its Python forms, and the packed format. No
GPU: a block of zeros stands for a handle (max_batch 0), since every refusal
comes before any device work."""
import ctypes

import pytest

import rlsampler

torch = pytest.importorskip("torch")
P = None
X = ctypes.c_void_p(64)  # an address that no refused call looks at


def weight(q=64, ldq=64, scale=64, lds=2, group=64):
    return rlsampler._Q4Weight(q, ldq, scale, lds, group)


def logits(h, hidden=X, ldh=128, w=None, B=0, H=128, V=10, out=X, dtype=0, ldo=10):
    return rlsampler.lib().rl_lmhead_q4_logits(h, hidden, ldh, w if w is not None else weight(), B, H, V, out, dtype, ldo, P)


def test_refusals():
    L, h = rlsampler.lib(), ctypes.create_string_buffer(4096)
    assert logits(None) == rlsampler.RL_ERR_INVALID_ARG and "handle" in rlsampler.last_error()
    assert L.rl_lmhead_q4_logits(h, X, 128, None, 0, 128, 10, X, 0, 10, P) == rlsampler.RL_ERR_INVALID_ARG
    assert L.rl_lmhead_q4_greedy(None, P, 128, weight(), 1, 128, 10, P, P, P, 10, P) == rlsampler.RL_ERR_INVALID_ARG
    assert L.rl_lmhead_q4_sample(None, P, 128, weight(), 1, 128, 10, P, P, 0, P, P, P, P, P, P) == rlsampler.RL_ERR_INVALID_ARG
    assert L.rl_lmhead_q4_quantize(None, X, 128, 128, 10, 64, X, 64, X, 2, P) == rlsampler.RL_ERR_INVALID_ARG
    assert logits(h) == rlsampler.RL_OK  # no rows: nothing to do
    for bad in (dict(B=-1), dict(H=0), dict(V=0), dict(ldh=120), dict(ldh=129), dict(ldo=9), dict(dtype=5), dict(hidden=ctypes.c_void_p(66)),
                dict(w=weight(q=72)), dict(w=weight(scale=65)), dict(w=weight(ldq=63)), dict(w=weight(ldq=72)), dict(w=weight(lds=1)),
                dict(B=1, hidden=P), dict(B=1, w=weight(q=None)), dict(B=1, w=weight(scale=None))):
        assert logits(h, **bad) == rlsampler.RL_ERR_INVALID_ARG, bad
        assert rlsampler.last_error(), bad
    for bad in (dict(w=weight(group=16)), dict(H=96, w=weight(group=32)), dict(H=192, ldh=192, w=weight(group=128, ldq=96))):
        assert logits(h, **bad) == rlsampler.RL_ERR_UNSUPPORTED, bad
    assert logits(h, B=1) == rlsampler.RL_ERR_SHAPE  # beyond max_batch
    assert L.rl_lmhead_q4_quantize(h, X, 127, 128, 10, 64, X, 64, X, 2, P) == rlsampler.RL_ERR_INVALID_ARG
    assert L.rl_lmhead_q4_quantize(h, X, 128, 128, 10, 48, X, 64, X, 2, P) == rlsampler.RL_ERR_UNSUPPORTED


def test_python_forms_refuse():
    q, s = torch.zeros(6, 64, dtype=torch.uint8), torch.zeros(6, 2, dtype=torch.bfloat16)
    rlsampler.Q4Weight(q, s, 64)
    for bad in ((q.int(), s, 64), (q, s.float(), 64), (q, s, 32), (q[:5], s, 64), (q.t(), s, 64)):
        with pytest.raises(ValueError):
            rlsampler.Q4Weight(*bad)
    sm = rlsampler.Sampler.__new__(rlsampler.Sampler)
    sm.h = None
    w = rlsampler.Q4Weight(q, s, 64)
    for bad in (torch.zeros(2, 128), torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(128, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            sm.lmhead_q4_logits(bad, w)
    with pytest.raises(ValueError):
        sm.lmhead_q4_logits(torch.zeros(2, 128, dtype=torch.bfloat16), w, out=torch.zeros(2, 7))
    for bad in ((torch.zeros(4, 96, dtype=torch.bfloat16), 32), (torch.zeros(4, 128, dtype=torch.bfloat16), 48),
                (torch.zeros(4, 128), 64), (torch.zeros(4, 192, dtype=torch.bfloat16), 128)):
        with pytest.raises(ValueError):
            sm.lmhead_q4_quantize(*bad)


def test_packed_format():
    codes = torch.arange(16, dtype=torch.uint8).repeat(1, 4)
    q = rlsampler.q4_pack(codes)
    # element 8 i + 2 j in bits 4 j of word i, element 8 i + 2 j + 1 in bits 16 + 4 j
    word = int.from_bytes(bytes(q[0, :4].tolist()), "little")
    assert [(word >> (4 * j)) & 15 for j in range(4)] == [0, 2, 4, 6]
    assert [(word >> (16 + 4 * j)) & 15 for j in range(4)] == [1, 3, 5, 7]
    assert torch.equal(rlsampler.q4_unpack(q), codes)
    r = torch.randint(0, 16, (5, 128))
    assert torch.equal(rlsampler.q4_unpack(rlsampler.q4_pack(r)), r.to(torch.uint8))
