"""How near the probabilities and draws of rl_specdec_verify_draft are to 64
bits, at rows where single precision alone would show."""
import numpy as np
import pytest

import rlsampler
from test_verify_draft_gpu import cuda

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LOG2E = np.log2(np.e)


@pytest.fixture(scope="module")
def smp():
    s = rlsampler.Sampler(0, max_batch=4, max_vocab=64, max_history=1)
    yield s
    s.close()


def hard_temperatures(rng, n):
    """Temperatures whose log2(e) / T lies furthest between two floats, in terms of itself."""
    T = rng.uniform(0.5, 1.5, 20000).astype(np.float32)
    c = LOG2E / T.astype(np.float64)
    off = np.abs(c.astype(np.float32) - c) / c
    return T[np.argsort(-off)[:n]]


@pytest.mark.parametrize("V", [600, 128256])
def test_probabilities_of_unlikely_tokens(smp, V):
    """An accepted token 50 binades below its row's largest. log2(e) / T as one
    float is off by up to 2^-24: 50 ln(2) 2^-24 in the probability. The weight is
    the product of two ex2 (2^-22 each); the sum has one more and is added up in
    floats over four levels (4 2^-24); the lane's and the warp's frames may move it
    (two ex2); the quotient is rounded once."""
    rng = np.random.default_rng(70)
    B = 48
    T = hard_temperatures(rng, B)
    x = (rng.normal(0, 1, (B, V)) - 8).astype(np.float32)
    x[:, 5] = rng.uniform(20, 30, B)
    at = rng.choice(np.arange(8, V), B)
    x[np.arange(B), at] = x[:, 5] - (50 * np.log(2.0) * T).astype(np.float32)
    rows = torch.from_numpy(np.repeat(x, 2, 0)).to(DEV)
    tok = cuda(at.astype(np.int32)[:, None])
    acc, out, prob, st = smp.specdec_verify_draft(rlsampler.DistRows(rows, cuda(T)), tok, torch.ones(B, dtype=torch.int32, device=DEV),
                                                  torch.zeros(B, 1, device=DEV), torch.full((B,), 0.5, device=DEV))
    assert (st == 0).all() and (acc == 1).all() and torch.equal(out[:, 0], tok[:, 0])
    z = x.astype(np.float64) / T.astype(np.float64)[:, None]
    p = np.exp(z[np.arange(B), at] - z[:, 5]) / np.exp(z - z[:, 5:6]).sum(1)
    off = np.abs(prob[:, 0].cpu().numpy() / p - 1)
    assert off.max() <= 50 * np.log(2.0) * 2.0 ** -24 + 5 * 2.0 ** -22 + 5 * 2.0 ** -24, off.max()


def rows_of(rng, kind, T, V):
    """Rows [len(T), V]: one id with half of the row and a tail of alike ids, or
    all within a few deviations of one another."""
    x = rng.normal(0, 0.3 if kind == "half" else 1.0, (len(T), V)).astype(np.float32)
    if kind == "half":
        for r, t in enumerate(T.astype(np.float64)):
            x[r, rng.integers(V // 4, 3 * V // 4)] = t * np.log(np.exp(x[r].astype(np.float64) / t).sum())
    return x


def draw(smp, x, T, u, row, drawn, z):
    """A token for each draw u of its row: of max(p - q, 0) behind a refused draft
    z that holds all of q, or of p."""
    B, K, R = len(u), 1 if drawn else 0, len(x)
    kw = {}
    if drawn:
        y = torch.full(x.shape, -np.inf, device=DEV)
        y[torch.arange(R, device=DEV), torch.from_numpy(z).to(DEV)] = 1.0
        kw["draft"] = rlsampler.DistRows(y, cuda(T[row]), first_row=cuda(row))
    acc, tok, prob, st = smp.specdec_verify_draft(
        rlsampler.DistRows(torch.from_numpy(np.repeat(x, K + 1, 0)).to(DEV), cuda(T[row]), first_row=cuda(row * (K + 1))),
        cuda(z[row].astype(np.int32)[:, None])[:, :K].contiguous(), torch.full((B,), K, dtype=torch.int32, device=DEV),
        torch.full((B, K), 0.999, device=DEV), cuda(u), **kw)
    assert (st == 0).all() and (acc == 0).all()
    return tok[:, 0].cpu().numpy()


def tolerance(w):
    """How far a running sum of a row of weights may be off, as a share of the
    whole. Ids of less than a sixteenth of a row are weighed in floats: an ex2
    (2^-22, which all may share: f (1 - f) of it where such ids are f of the row) and
    an exponent rounded twice (2^-20 of each weight together, at exponents up to 32;
    independent, so that eight deviations of the sum are 8 2^-20 sqrt(sum of squares))."""
    light = w[w < w.sum() / 16] / w.sum()
    return light.sum() * (1 - light.sum()) * 2.0 ** -22 + 8 * 2.0 ** -20 * np.sqrt((light ** 2).sum()) + 1e-10


@pytest.mark.parametrize("kind", ["half", "flat"])
@pytest.mark.parametrize("drawn", [False, True])
def test_draws_next_to_borders(smp, kind, drawn):
    """Draws that lie one to two tolerances from a running sum's border give the
    id that 64 bits give."""
    rng = np.random.default_rng(71 + drawn)
    V, R, each = 128256, 5, 100
    T = hard_temperatures(rng, R)
    x = rows_of(rng, kind, T, V)
    z = rng.choice(V, R)
    us, want = [], []
    for r in range(R):
        w = np.exp((x[r].astype(np.float64) - x[r].max()) / T[r].astype(np.float64))
        if drawn:
            w[z[r]] = 0.0
        run = np.cumsum(w) / w.sum()
        tol = tolerance(w)
        assert tol < 1.5e-7
        j = rng.permutation(np.flatnonzero((run > 0.05) & (run < 0.95)))
        u = (run[j] + rng.choice([-1.5, 1.5], len(j)) * tol).astype(np.float32)
        off = np.abs(u.astype(np.float64)[:, None] - run[np.clip(j[:, None] + np.arange(-3, 4), 0, V - 1)]).min(1)
        u = u[(off > tol) & (off < 2 * tol)][:each]
        assert len(u) == each
        us.append(u)
        want.append((run[None, :] <= u.astype(np.float64)[:, None]).sum(1))
    u, want = np.concatenate(us), np.concatenate(want)
    tok = draw(smp, x, T, u, np.repeat(np.arange(R, dtype=np.int32), each), drawn, z)
    assert np.array_equal(tok, want), (np.flatnonzero(tok != want).size, len(u))


@pytest.mark.parametrize("drawn", [False, True])
def test_light_ids_beside_a_heavy_one(smp, drawn):
    """One id holds nearly all of a row, the others 4e-8 of it each. Added to that id
    in floats the ids beside it would vanish, and every running sum behind it be
    short by up to 15 of them (6e-7); the tolerance is 2e-9."""
    rng = np.random.default_rng(73 + drawn)
    V, R, each = 128256, 6, 80
    T = hard_temperatures(rng, R)
    x = (rng.normal(0, 0.3, (R, V)) * T[:, None]).astype(np.float32)
    z = rng.integers(100, 2000, R)
    us, want = [], []
    for r in range(R):
        top = 512 * 40 + 4 * int(rng.integers(0, 32))
        x[r, top] = np.float32(17.0 * T[r])
        w = np.exp((x[r].astype(np.float64) - x[r, top]) / T[r].astype(np.float64))
        if drawn:
            w[z[r]] = 0.0
        run = np.cumsum(w) / w.sum()
        tol = tolerance(w)
        assert tol < 2.5e-9 and 1 - run[top] > 1e-3
        u = np.unique((run[32768] + (1 - run[32768]) * rng.random(4 * each)).astype(np.float32))
        u = u[u < run[V - 100]]
        at = np.searchsorted(run, u.astype(np.float64), side="right")
        off = np.minimum(run[at] - u, u - run[at - 1])
        u, at = u[off > tol][:each], at[off > tol][:each]
        assert len(u) == each
        us.append(u)
        want.append(at)
    u, want = np.concatenate(us), np.concatenate(want)
    tok = draw(smp, x, T, u, np.repeat(np.arange(R, dtype=np.int32), each), drawn, z)
    assert np.array_equal(tok, want), (np.flatnonzero(tok != want).size, len(u))
