"""The LM head with 4-bit weights (rl_lmhead_q4_*) against float64 products of
the same codes, scales and bf16 hidden states.

Tolerance: code - 8 times a bf16 value is exact in f32, so a logit is an f32
sum of H exact terms (in whatever order, each addition off by at most 2^-23 of
its result where the tensor cores truncate) with one more rounding for each
group's scale and sum: at most H * 2^-22 * sum |terms|.
"""
import numpy as np
import pytest

import oracle
import rlsampler
import workloads

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def smp():
    s = rlsampler.Sampler(0, max_batch=600, max_vocab=40000, max_history=64)
    yield s
    s.close()


def make(B, H, V, G, seed, pad_q=0, pad_s=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hidden = torch.randn(B, H, generator=g, device="cuda").to(torch.bfloat16)
    codes = torch.randint(0, 16, (V, H), generator=g, device="cuda")
    q = torch.full((V, H // 2 + pad_q), 0xEE, dtype=torch.uint8, device="cuda")[:, : H // 2]
    q.copy_(rlsampler.q4_pack(codes))
    scale = torch.full((V, H // G + pad_s), float("nan"), dtype=torch.bfloat16, device="cuda")[:, : H // G]
    scale.copy_((torch.rand(V, H // G, generator=g, device="cuda") + 0.1) * H ** -0.5)
    scale[::3] *= -1
    return hidden, codes, rlsampler.Q4Weight(q, scale, G)


def exact(hidden, codes, w):
    dense = ((codes.double() - 8).view(w.V, -1, w.group) * w.scale.double()[:, :, None]).flatten(1)
    h = hidden.double()
    return h @ dense.T, h.abs() @ dense.abs().T


def check(hidden, codes, w, got):
    ref, mag = exact(hidden, codes, w)
    err = (got.double() - ref).abs()
    bound = hidden.shape[1] * 2.0 ** -22 * mag + 1e-30
    assert bool((err <= bound).all()), f"max err {err.max().item():.3e}, bound there {bound.flatten()[err.argmax()].item():.3e}"


SHAPES = [(1, 64, 1, 32), (1, 64, 2, 64), (3, 128, 127, 128), (1, 128, 128, 32), (2, 192, 129, 64), (5, 192, 300, 32),
          (1, 256, 1000, 128), (7, 320, 1000, 64), (8, 512, 1111, 128), (9, 1024, 5000, 32), (16, 2048, 3000, 64),
          (17, 2048, 3001, 128), (31, 448, 777, 64), (32, 512, 2000, 32), (33, 512, 2000, 128), (48, 1024, 1500, 32),
          (49, 640, 900, 128), (64, 4096, 4000, 32), (65, 576, 900, 64), (96, 1024, 1300, 64), (97, 1024, 1300, 128),
          (128, 2048, 2222, 128), (129, 512, 700, 64), (256, 512, 1000, 32), (257, 256, 500, 128), (600, 128, 300, 64),
          (1, 4096, 32000, 128), (12, 6144, 20001, 32), (1, 16384, 3000, 64)]


@pytest.mark.parametrize("B,H,V,G", SHAPES)
def test_logits(smp, B, H, V, G):
    hidden, codes, w = make(B, H, V, G, B + H + V)
    got = smp.lmhead_q4_logits(hidden, w)
    torch.cuda.synchronize()
    check(hidden, codes, w, got)


@pytest.mark.parametrize("B,H,V,G", [(1, 256, 1000, 32), (20, 512, 3001, 128), (100, 192, 515, 64)])
def test_bf16_logits_are_rounded_f32_logits(smp, B, H, V, G):
    hidden, codes, w = make(B, H, V, G, 5)
    f = smp.lmhead_q4_logits(hidden, w)
    b = smp.lmhead_q4_logits(hidden, w, out_dtype=torch.bfloat16)
    torch.cuda.synchronize()
    assert torch.equal(b.view(torch.int16), f.to(torch.bfloat16).view(torch.int16))


@pytest.mark.parametrize("B,V,pad_q,pad_s,pad_o", [(1, 300, 16, 1, 3), (5, 1001, 48, 5, 0), (40, 515, 32, 3, 7), (130, 260, 16, 8, 1)])
def test_strides(smp, B, V, pad_q, pad_s, pad_o):
    H, G = 384, 64
    hidden, codes, w = make(B, H, V, G, 6, pad_q, pad_s)
    wide = torch.full((B, H + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, :H] = hidden
    buf = torch.full((B, V + pad_o), 7.0, device="cuda")
    smp.lmhead_q4_logits(wide[:, :H], w, out=buf[:, :V])
    torch.cuda.synchronize()
    check(hidden, codes, w, buf[:, :V])
    assert bool((buf[:, V:] == 7.0).all())


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1e6, 1e30])
def test_scales_of_any_size(smp, scale):
    hidden, codes, w = make(4, 256, 400, 32, 8)
    w.scale.mul_(scale)
    w.scale[5, 2], w.scale[6] = 0.0, 0.0
    got = smp.lmhead_q4_logits(hidden, w)
    torch.cuda.synchronize()
    check(hidden, codes, w, got)
    assert bool((got[:, 6] == 0).all())


@pytest.mark.parametrize("B", [3, 40])
def test_nonfinite_values_stay_in_their_rows(smp, B):
    hidden, codes, w = make(B, 256, 400, 64, 9)
    good = smp.lmhead_q4_logits(hidden, w)
    hidden[1, 17], w.scale[7, 1] = float("nan"), float("nan")
    hidden[2, 5] = float("inf")
    got = smp.lmhead_q4_logits(hidden, w)
    torch.cuda.synchronize()
    assert bool(got[1].isnan().all()) and bool(got[:, 7].isnan().all())
    assert not bool(got[2].isfinite().any())
    rest = [b for b in range(B) if b not in (1, 2)]
    cols = [v for v in range(400) if v != 7]
    assert torch.equal(got[rest][:, cols], good[rest][:, cols])


@pytest.mark.parametrize("B,H,V,G", [(1, 64, 1, 32), (3, 256, 1000, 64), (17, 1024, 5000, 128), (64, 512, 3000, 32),
                                     (128, 256, 2001, 128), (300, 128, 700, 64)])
def test_greedy_matches_own_logits(smp, B, H, V, G):
    hidden, codes, w = make(B, H, V, G, 3 * B + V)
    lg = torch.empty(B, V, device="cuda")
    tok, st = smp.lmhead_q4_greedy(hidden, w, out_logits=lg)
    tok2, st2 = smp.lmhead_q4_greedy(hidden, w)
    torch.cuda.synchronize()
    check(hidden, codes, w, lg)
    x = lg.cpu().numpy()
    want = np.array([oracle.greedy(x[b]) for b in range(B)], np.int32)
    assert (st.cpu().numpy() == 0).all() and (st2.cpu().numpy() == 0).all()
    assert np.array_equal(tok.cpu().numpy(), want) and np.array_equal(tok2.cpu().numpy(), want)


@pytest.mark.parametrize("B", [4, 70])
def test_greedy_ties_take_the_last_maximum(smp, B):
    hidden, codes, w = make(B, 128, 1000, 64, 9)
    hidden = hidden.abs()
    codes[[5, 77, 300, 611]] = 15
    w.scale[[5, 77, 300, 611]] = 4.0
    w = rlsampler.Q4Weight(rlsampler.q4_pack(codes), w.scale.contiguous(), 64)
    tok, st = smp.lmhead_q4_greedy(hidden, w)
    torch.cuda.synchronize()
    assert tok.cpu().tolist() == [611] * B and st.cpu().tolist() == [0] * B


def test_sample_equals_sampler_on_own_logits(smp):
    B, H, V = 48, 512, 32000
    hidden, _, w = make(B, H, V, 128, 11)
    r = np.random.default_rng(11)
    p = np.zeros(B, rlsampler.ROW_PARAMS_DTYPE)
    p["temperature"], p["top_k"], p["top_p"] = r.uniform(0.5, 1.5, B), r.choice([0, 1, 20, 50], B), r.uniform(0.8, 1.0, B)
    p["repeat_penalty"] = r.uniform(1.0, 1.3, B)
    hist = torch.from_numpy(r.integers(0, V, (B, 64)).astype(np.int32)).cuda()
    hl = torch.from_numpy(r.integers(0, 65, B).astype(np.int32)).cuda()
    u = torch.from_numpy(workloads.uniforms(9, 0, B)).cuda()
    pd = rlsampler.params_tensor(p, "cuda")
    got = smp.lmhead_q4_sample(hidden, w, pd, u, hist, hl)
    want = smp.sample(smp.lmhead_q4_logits(hidden, w), pd, u, hist, hl)
    torch.cuda.synchronize()
    for g, x in zip(got, want):
        assert torch.equal(g, x)
    assert (got[2].cpu().numpy() == 0).all()


def reference_codes(w, G):
    """Codes and scales by the definition, in torch (elementwise f32, IEEE)."""
    V, H = w.shape
    x = w.float().view(V, H // G, G)
    at = x.abs().argmax(2, keepdim=True)  # replaced below by the first of equals
    top = x.abs().amax(2, keepdim=True)
    ids = torch.arange(G, device=w.device)
    at = torch.where(x.abs() == top, ids, G).amin(2, keepdim=True).clamp(max=G - 1)
    s = (-x.gather(2, at) / 8).to(torch.bfloat16)
    s = torch.where(s == 0, torch.zeros_like(s), s)
    c = torch.clamp(torch.round(x / s.float()) + 8, 0, 15)
    c = torch.where(s == 0, torch.full_like(c, 8), c)
    bad = ~x.isfinite().all(2, keepdim=True)
    c = torch.where(bad, torch.full_like(c, 8), c)
    s = torch.where(bad, torch.full_like(s, float("nan")), s)
    return c.view(V, H).to(torch.uint8), s[:, :, 0]


@pytest.mark.parametrize("V,H,G", [(1, 64, 32), (3, 64, 64), (7, 128, 128), (129, 192, 64), (1000, 1024, 32), (517, 2560, 128),
                                   (4000, 4096, 64)])
@pytest.mark.parametrize("size", [0.02, 1.0, 1e-30, 1e20])
def test_quantize_bit_for_bit(smp, V, H, G, size):
    g = torch.Generator(device="cuda").manual_seed(V + H)
    x = (torch.randn(V, H + 8, generator=g, device="cuda") * size).to(torch.bfloat16)[:, :H]
    x[0, :32] = 0.0
    if V > 2:
        x[1] = torch.round(torch.randn(H, generator=g, device="cuda") * 2).to(torch.bfloat16)  # ties of both signs, halves
        x[2, 3], x[2, H - 1] = float("nan"), float("inf")
    w = smp.lmhead_q4_quantize(x, G)
    torch.cuda.synchronize()
    c, s = reference_codes(x, G)
    assert torch.equal(rlsampler.q4_unpack(w.q), c)
    assert torch.equal(w.scale.view(torch.int16)[~s.isnan()], s.view(torch.int16)[~s.isnan()])
    assert torch.equal(w.scale.isnan(), s.isnan())
    # a step is the scale: every weight within half of one, the far end within one
    back = (c.double() - 8).view(V, -1, G) * s.double()[:, :, None]
    err = (back - x.double().view(V, -1, G)).abs() / s.double().abs()[:, :, None].clamp(min=1e-300)
    ok = s.isfinite() & (s != 0)
    assert float(err[ok].max()) <= 1.0 + 1e-9


def test_quantized_head_follows_the_bf16_head(smp):
    """bf16 weights, quantised and multiplied: the 64-bit product of the
    quantised weights, and near the bf16 head's logits (a weight is off by at
    most one step, top / 8, of its group: the mean square error of a logit over
    rows is below that of steps, H (top / 8)^2 / 12, by a factor of the number
    of standard deviations of the top)."""
    g = torch.Generator(device="cuda").manual_seed(3)
    hidden = torch.randn(24, 1024, generator=g, device="cuda").to(torch.bfloat16)
    weight = (torch.randn(3000, 1024, generator=g, device="cuda") / 32).to(torch.bfloat16)
    w = smp.lmhead_q4_quantize(weight, 32)
    got = smp.lmhead_q4_logits(hidden, w)
    full = smp.lmhead_logits(hidden, weight)
    torch.cuda.synchronize()
    check(hidden, rlsampler.q4_unpack(w.q), w, got)
    rms = (got - full).pow(2).mean().sqrt().item()
    assert 0 < rms < (weight.float().abs().max().item() / 8) * 1024 ** 0.5


def test_graphs_and_another_stream(smp):
    hidden, codes, w = make(9, 512, 2000, 64, 21)
    want = smp.lmhead_q4_logits(hidden, w)
    tok, _ = smp.lmhead_q4_greedy(hidden, w)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = smp.lmhead_q4_logits(hidden, w)
    s.synchronize()
    assert torch.equal(got, want)
    out, g = torch.zeros_like(want), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        smp.lmhead_q4_logits(hidden, w, out=out)
        t2, _ = smp.lmhead_q4_greedy(hidden, w)
    for _ in range(2):
        out.zero_()
        t2.fill_(-7)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(t2, tok)
    del g


def test_repeated_calls_give_the_same_bits(smp):
    hidden, codes, w = make(33, 1024, 5000, 32, 22)
    a = smp.lmhead_q4_logits(hidden, w)
    for _ in range(3):
        assert torch.equal(a, smp.lmhead_q4_logits(hidden, w))


def test_argument_errors(smp):
    hidden, _, w = make(4, 128, 300, 64, 1)
    with pytest.raises(ValueError):
        smp.lmhead_q4_logits(hidden[:, :64], w)
    with pytest.raises(ValueError):
        smp.lmhead_q4_logits(hidden, w, out=torch.empty(4, 299, device="cuda"))
    with pytest.raises(rlsampler.RLError) as e:
        smp.lmhead_q4_logits(torch.empty(601, 128, dtype=torch.bfloat16, device="cuda"), w)
    assert e.value.status == rlsampler.RL_ERR_SHAPE
    odd = torch.empty(4, 136, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(rlsampler.RLError) as e:
        smp.lmhead_q4_logits(odd[:, 1:129], w)
    assert e.value.status == rlsampler.RL_ERR_INVALID_ARG
    with pytest.raises(rlsampler.RLError) as e:  # vocabulary beyond the handle's
        _, _, big = make(1, 64, 40001, 64, 2)
        smp.lmhead_q4_sample(torch.empty(1, 64, dtype=torch.bfloat16, device="cuda"), big, torch.zeros(24, dtype=torch.uint8, device="cuda"),
                             torch.zeros(1, device="cuda"))
    assert e.value.status == rlsampler.RL_ERR_SHAPE


@pytest.mark.parametrize("B", [3, 40])
def test_offsets_past_32_bits(smp, B):
    """Codes and scales of the last rows lie beyond 2^32 bytes; logits too."""
    H, V, G = 256, 70, 64
    hidden, codes, w = make(B, H, V, G, 41)
    ldq, lds = 1 << 26, (1 << 25) + 8
    q = torch.empty(V * ldq, dtype=torch.uint8, device="cuda").as_strided((V, H // 2), (ldq, 1))
    s = torch.empty(V * lds, dtype=torch.bfloat16, device="cuda").as_strided((V, H // G), (lds, 1))
    q.copy_(w.q)
    s.copy_(w.scale)
    want = smp.lmhead_q4_logits(hidden, w)
    got = smp.lmhead_q4_logits(hidden, rlsampler.Q4Weight(q, s, G))
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    del q, s
    ldo = (1 << 30) + 1 if B < 8 else 1 << 27
    out = torch.empty(B * ldo, dtype=torch.float32, device="cuda").as_strided((B, V), (ldo, 1))
    smp.lmhead_q4_logits(hidden, w, out=out)
    assert torch.equal(out, want)


@pytest.mark.parametrize("B", [4, 30])
@pytest.mark.parametrize("H,G", [(256, 32), (512, 64), (1024, 128), (256, 128)])
@pytest.mark.parametrize("lead,pad", [(0, 0), (1, 0), (2, 2), (4, 4), (0, 1), (8, 8)])
def test_scales_on_any_boundary(smp, B, H, G, lead, pad):
    """Scales that start at any element and at any row stride."""
    V = 333
    hidden, codes, w = make(B, H, V, G, 42)
    n = H // G
    buf = torch.full((lead + V * (n + pad),), float("nan"), dtype=torch.bfloat16, device="cuda")
    s = buf[lead:].as_strided((V, n), (n + pad, 1), lead)
    s.copy_(w.scale)
    got = smp.lmhead_q4_logits(hidden, rlsampler.Q4Weight(w.q, s, G))
    assert torch.equal(got, smp.lmhead_q4_logits(hidden, w))
