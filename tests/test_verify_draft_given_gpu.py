"""Given drafts (no draft distribution) under masks and cutoffs, up to siblings
that cover all that a row keeps. Tolerances as in test_verify_draft_gpu.py."""
import numpy as np
import pytest

import rlsampler
from test_verify_draft_gpu import Case, TREES, cuda

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BELOW_1 = np.nextafter(np.float32(1), np.float32(0))


@pytest.fixture(scope="module")
def smp():
    s = rlsampler.Sampler(0, max_batch=4, max_vocab=64, max_history=1)
    yield s
    s.close()


def likely(c, rng, most=4):
    """Children that are likely by the target's own rows; siblings may repeat."""
    for b in range(c.B):
        for i in range(1, c.N):
            src = c.parent[b, i] if c.tree else i - 1
            x = c.x[b * c.N + src].copy()
            if c.mask is not None and c.mask[b * c.N + src].any():
                bits = np.unpackbits(c.mask[b * c.N + src].view(np.uint8), bitorder="little")[: c.V].astype(bool)
                x[~bits] = -np.inf
            t = np.argsort(-x)[min(c.V - 1, int(rng.integers(0, most)))]
            if c.tree:
                c.tok[b, i] = t
            else:
                c.tok[b, i - 1] = t


@pytest.mark.parametrize("mask,cut", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("V,lead", [(40, 0), (1001, 3), (32000, 0)])
def test_chain_masks_and_cutoffs(smp, mask, cut, V, lead):
    rng = np.random.default_rng(V + 2 * mask + cut)
    c = Case(rng, 16, V, K=3, mask=mask, cut=cut, lead=lead, draft=False, sigma=2.0)
    likely(c, rng, 2)
    # how many are accepted is the inputs' business: the largest of 32,000 masked
    # normal logits of deviation 2 has about e^8 / (16,000 e^2) = 2.5% of its row
    c.check(c.call(smp))


@pytest.mark.parametrize("shape", ["2", "3.1", "4.2.1", "late"])
@pytest.mark.parametrize("mask,cut", [(True, False), (False, True), (True, True)])
def test_tree_masks_and_cutoffs(smp, shape, mask, cut):
    rng = np.random.default_rng(len(shape) + 2 * mask + cut)
    c = Case(rng, 40, 300, parents=TREES[shape], mask=mask, cut=cut, draft=False, sigma=2.0)
    likely(c, rng)
    assert c.check(c.call(smp)).max() > 0


def covered(rng, kept, how, V=3000, B=64, share=None):
    """Trees whose root has `kept` children: all that its row keeps."""
    c = Case(rng, B, V, parents=[-1] + [0] * kept, draft=False, sigma=1.0)
    N = kept + 1
    sets = np.stack([rng.choice(V, kept, replace=False) for _ in range(B)])
    for b in range(B):
        r = b * N
        if share is not None:  # these shares of the kept ids, the largest first
            c.x[r, :] = -50.0
            c.x[r, sets[b]] = np.log(share[b]).astype(np.float32)
        if how == "cut":  # the kept ids above all others (with shares: every id alike, and the kept ones in order up to the cutoff)
            c.x[r, :] = np.minimum(c.x[r], 3.0 if share is None else -50.0)
            if share is None:
                c.x[r, sets[b]] = 4.0 + rng.random(kept).astype(np.float32) * 3
        c.tok[b, 1:] = sets[b]
    c.pr.copy_(torch.from_numpy(c.x))
    if how == "mask":
        c.mask = np.zeros((B * N, (V + 31) // 32), np.uint32)
        for b in range(B):
            for t in sets[b]:
                c.mask[b * N, t >> 5] |= np.uint32(1 << (t & 31))
    else:
        c.cut = np.full(B * N, -1, np.int32)
        for b in range(B):
            best = min(sets[b], key=lambda t: (c.x[b * N, t], -t))  # the last one kept
            c.cut[b * N] = best
    return c, sets


@pytest.mark.parametrize("kept", [1, 2, 5])
@pytest.mark.parametrize("how", ["mask", "cut"])
@pytest.mark.parametrize("u", [1.0, BELOW_1, 0.97])
def test_siblings_that_cover_what_is_kept(smp, kept, how, u):
    """Every sequence that ends well gets a kept token, also where all were refused."""
    rng = np.random.default_rng(60 + kept)
    c, sets = covered(rng, kept, how)
    c.u[:] = u
    out = c.call(smp)
    acc, path, tok, prob, st = out
    assert (st == 0).all()
    # (with u = 1 the last one left stands at its border, u sum(w) = w(x) in exact
    # numbers, where both sides' roundings decide: either way is right)
    for b in range(c.B):
        assert tok[b, 0] in sets[b] and prob[b, 0] > 0, (b, tok[b], sets[b])
        if acc[b] == 0:
            assert (path[b] == -1).all() and (tok[b, 1:] == -1).all(), b
    if u < BELOW_1:
        c.check(out)
        assert acc.max() == 1


@pytest.mark.parametrize("how", ["mask", "cut", "cut behind the shares"])
@pytest.mark.parametrize("rest", [1e-3, 1e-5, 2e-7])
def test_small_rest_behind_a_refused_sibling(smp, how, rest):
    """All but `rest` of a row on its first child, which is refused: the others
    are accepted by their shares of the rest, as in 64 bits."""
    rng = np.random.default_rng(61)
    B, kept = 256, 4
    part = rng.dirichlet(np.full(kept - 1, 2.0), B) * rest
    c, sets = covered(rng, kept, how, B=B, share=np.concatenate([np.full((B, 1), 1.0 - rest), part], 1))
    c.u[:, 1] = 2.0  # refused, and far from its border
    c.u[:, 2:] = rng.random((B, kept - 1)).astype(np.float32)
    out = c.call(smp)
    c.check(out)
    if how != "cut":
        assert 0 < out[0].mean() <= 1
