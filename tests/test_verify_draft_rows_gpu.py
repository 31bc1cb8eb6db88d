"""rl_specdec_verify_tree over packed draft rows: which rows a sequence may have."""
import numpy as np
import pytest

import rlsampler
from test_verify_draft_gpu import Case, cuda

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def smp():
    s = rlsampler.Sampler(0, max_batch=4, max_vocab=64, max_history=1)
    yield s
    s.close()


@pytest.mark.parametrize("nowhere", ["behind", "before", "far"])
def test_a_root_alone_has_no_draft_row(smp, nowhere):
    """Trees of their root only among others, with packed draft rows and cutoffs:
    the root's first_row names no row (the end of the array, -1, far away), none
    is read, and the token is the one that a call without draft rows gives."""
    rng = np.random.default_rng(50)
    B, V, N = 12, 200, 4
    c = Case(rng, B, V, parents=[-1, 0, 0, 1], cut=True)
    c.n[::3] = 1
    want = c.call(smp)
    keep = np.concatenate([np.arange(b * N, b * N + N) for b in range(B) if c.n[b] > 1])
    first = np.zeros(B, np.int32)
    first[c.n > 1] = np.arange((c.n > 1).sum()) * N
    first[c.n == 1] = {"behind": len(keep), "before": -1, "far": 2 ** 31 - 8}[nowhere]
    t = rlsampler.DistRows(c.pr, cuda(c.T), cut=cuda(c.cut))
    d = rlsampler.DistRows(c.qr[torch.from_numpy(keep).to(DEV)].contiguous(), cuda(c.Tq), cut=cuda(c.qcut[keep]), first_row=cuda(first))
    got = smp.specdec_verify_tree(t, cuda(c.tok), cuda(c.parent), cuda(c.n), cuda(c.u), cuda(c.du), draft=d)
    for g, w in zip(got, want):
        assert np.array_equal(g.cpu().numpy(), w)


def test_no_draft_rows_at_all(smp):
    """Every tree is a root alone: the draft may have no rows (and no address)."""
    rng = np.random.default_rng(51)
    B, V, N = 6, 130, 3
    c = Case(rng, B, V, parents=[-1, 0, 0], cut=True)
    c.n[:] = 1
    want = c.call(smp)
    d = rlsampler.DistRows(torch.empty(0, V, device=DEV), cuda(c.Tq), cut=torch.empty(0, dtype=torch.int32, device=DEV),
                           first_row=torch.zeros(B, dtype=torch.int32, device=DEV))
    got = smp.specdec_verify_tree(rlsampler.DistRows(c.pr, cuda(c.T), cut=cuda(c.cut)), cuda(c.tok), cuda(c.parent), cuda(c.n),
                                  cuda(c.u), cuda(c.du), draft=d)
    for g, w in zip(got, want):
        assert np.array_equal(g.cpu().numpy(), w)


@pytest.mark.parametrize("which", ["draft", "target", "both"])
@pytest.mark.parametrize("parents", [None, [-1, 0, 0, 1, 1, 2]])
def test_masks_without_a_bit(smp, which, parents):
    """A mask row without a bit allows every id, on either side, at any node."""
    rng = np.random.default_rng(52)
    B, V = 24, 700
    c = Case(rng, B, V, parents=parents, K=None if parents else 4, mask=True, noise=1.5)
    if which != "target":
        c.qmask[rng.random(len(c.qmask)) < 0.6] = 0
    if which != "draft":
        c.mask[rng.random(len(c.mask)) < 0.6] = 0
    c.check(c.call(smp))
