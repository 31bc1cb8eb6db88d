"""rl_specdec_verify_draft and rl_specdec_verify_tree against the 64-bit
restatement (oracle/verify.py).

Tolerance. A weight 2^((x - m) c) in f32 has a relative error of at most
2^-22 (ex2) + |t| 2^-23 (the rounding of x - m and of the products, t <= 64 for
any weight that matters) < 2^-16, and typically 2^-22; a sum of weights has the
largest of its terms' errors. So probabilities, accept tests and running sums
are off by at most EPS = 2^-16 of the row's whole mass (times 1 + C for
residuals, C <= the number of siblings). Decisions further than that from
their border have to agree; a drawn token has to be the one whose running sums
enclose the target up to EPS. Most rows are compared more tightly: all but a
few tokens have to be equal outright.
"""
import numpy as np
import pytest

import rlsampler
import verify as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 2.0 ** -16


@pytest.fixture(scope="module")
def smp():
    s = rlsampler.Sampler(0, max_batch=4, max_vocab=64, max_history=1)
    yield s
    s.close()


def cuda(x):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to(DEV)


def rows(x, dtype, pad=0, lead=0):
    """[R, V] on the device at row stride V + pad, `lead` elements behind an aligned address."""
    t = torch.float32 if dtype == "f32" else torch.bfloat16
    R, V = x.shape
    buf = torch.full((lead + R * (V + pad),), 5.0, dtype=t, device=DEV)
    v = buf[lead:].view(R, V + pad)[:, :V]
    v.copy_(torch.from_numpy(x))
    return v


class Case:
    """B chains or trees with what the call and the restatement need."""

    def __init__(self, rng, B, V, parents=None, K=None, pd="f32", qd="f32", pad=0, lead=0, mask=False, cut=False,
                 draft=True, T=None, sigma=3.0, noise=0.6):
        self.tree = parents is not None
        self.B, self.V = B, V
        self.N = N = len(parents) if self.tree else K + 1
        self.Q = N if self.tree else K
        x = (rng.normal(0, sigma, (B * N, V))).astype(np.float32)
        y = (0.95 * x + rng.normal(0, noise, x.shape)).astype(np.float32)
        y = y.reshape(B, N, V)[:, : self.Q].reshape(B * self.Q, V)
        self.pr, self.qr = rows(x, pd, pad, lead), rows(y, qd, pad, lead) if draft else None
        self.x = self.pr.float().cpu().numpy()
        self.y = self.qr.float().cpu().numpy() if draft else y
        self.T = np.full(B, 1.0, np.float32) if T is None else np.asarray(T, np.float32)
        self.Tq = self.T.copy()
        self.parent = np.tile(np.asarray(parents, np.int32), (B, 1)) if self.tree else None
        self.n = np.full(B, N if self.tree else K, np.int32)
        self.mask = self.qmask = self.cut = self.qcut = None
        W = (V + 31) // 32
        if mask:
            self.mask = rng.integers(0, 2 ** 32, (B * N, W), dtype=np.uint32) | rng.integers(0, 2 ** 32, (B * N, W), dtype=np.uint32)
            self.mask[:: 3] = 0
            self.qmask = rng.integers(0, 2 ** 32, (B * self.Q, W), dtype=np.uint32)
        if cut:
            self.cut = np.argsort(-self.x, 1, kind="stable")[np.arange(B * N), rng.integers(0, min(V, 40), B * N)].astype(np.int32)
            self.cut[::5] = -2
            self.qcut = np.argsort(-self.y, 1, kind="stable")[np.arange(B * self.Q), rng.integers(0, min(V, 40), B * self.Q)].astype(np.int32) if self.Q else None
        self.u = rng.random((B, N if self.tree else K)).astype(np.float32)
        self.du = rng.random(B).astype(np.float32)
        tok = np.zeros((B, N), np.int32)
        for b in range(B):
            for i in range(1, N):
                src = self.parent[b, i] if self.tree else i - 1
                q = ref.dist(self.y[b * self.Q + src], max(self.Tq[b], 0.3), self.row(self.qmask, b * self.Q + src),
                             self.row(self.qcut, b * self.Q + src))
                tok[b, i] = rng.choice(V, p=q)
        self.tok = tok if self.tree else tok[:, 1:].copy()

    @staticmethod
    def row(a, r):
        return None if a is None else a[r]

    def call(self, smp, stream=None):
        i32 = lambda m: None if m is None else cuda(m.view(np.int32))  # noqa: E731
        t = rlsampler.DistRows(self.pr, cuda(self.T), i32(self.mask), cuda(self.cut))
        d = None if self.qr is None else rlsampler.DistRows(self.qr, cuda(self.Tq), i32(self.qmask), cuda(self.qcut))
        if self.tree:
            out = smp.specdec_verify_tree(t, cuda(self.tok), cuda(self.parent), cuda(self.n), cuda(self.u), cuda(self.du), draft=d, stream=stream)
        else:
            acc, tk, pr, st = smp.specdec_verify_draft(t, cuda(self.tok), cuda(self.n), cuda(self.u), cuda(self.du), draft=d, stream=stream)
            path = torch.arange(1, tk.shape[1] + 1, device=DEV).repeat(tk.shape[0], 1).int()
            out = acc, path.masked_fill(path > acc[:, None], -1), tk, pr, st
        torch.cuda.synchronize()
        return [o.cpu().numpy() for o in out]

    def walk(self, b):
        N, Q, T = self.N, self.Q, float(self.T[b])
        n = int(self.n[b]) + (0 if self.tree else 1)

        def q_of(i):
            if self.qr is None or self.Tq[b] <= 0:
                return None
            q = ref.dist(self.y[b * Q + i], float(self.Tq[b]), self.row(self.qmask, b * Q + i), self.row(self.qcut, b * Q + i))
            return "bad" if q is None else q

        return ref.walk(lambda i: ref.dist(self.x[b * N + i], T, self.row(self.mask, b * N + i), self.row(self.cut, b * N + i)),
                        q_of, (lambda i: [c for c in range(i + 1, n) if self.parent[b, c] == i]) if self.tree else (lambda i: [i + 1] if i + 1 < n else []),
                        (lambda c: int(self.tok[b, c])) if self.tree else (lambda c: int(self.tok[b, c - 1])),
                        (lambda c: self.u[b, c]) if self.tree else (lambda c: self.u[b, c - 1]), self.du[b], greedy=T <= 0)

    def check(self, out, ok=0.98):
        acc, path, tok, prob, st = out
        same = 0
        for b in range(self.B):
            r = self.walk(b)
            if r.bad:
                assert st[b] == rlsampler.RL_ERR_NONFINITE and acc[b] == -1 and (tok[b] == -1).all() and (prob[b] == 0).all(), b
                assert (path[b] == -1).all()
                same += 1
                continue
            assert st[b] == 0, (b, st[b])
            if r.accept_margin < EPS:
                same += 1
                continue  # a test within the rounding: either way is right
            k = len(r.path)
            assert acc[b] == k, (b, acc[b], r.path)
            assert path[b, :k].tolist() == r.path and (path[b, k:] == -1).all()
            assert tok[b, :k].tolist() == r.tokens[:k] and (tok[b, k + 1:] == -1).all()
            x = int(tok[b, k])
            tol = EPS * (1 + self.N)
            assert 0 <= x < self.V and r.p[x] > 0, (b, x)
            lo = r.run[x - 1] if x else 0.0
            assert lo - tol <= r.target <= r.run[x] + tol, (b, x, lo, r.target, r.run[x])
            want = np.array(r.probs[:k] + [r.p[x]])
            # Z and the weight each within the weights' relative error
            np.testing.assert_allclose(prob[b, : k + 1], want, rtol=2 * EPS, atol=1e-37)
            assert (prob[b, k + 1:] == 0).all()
            same += x == r.tokens[-1]
        assert same >= ok * self.B - 1, (same, self.B)
        return acc


@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 31, 33, 255, 1000, 4099])
@pytest.mark.parametrize("pd,qd", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
def test_chain_sizes_and_types(smp, V, pd, qd):
    rng = np.random.default_rng(V)
    c = Case(rng, 40, V, K=4, pd=pd, qd=qd, T=rng.uniform(0.5, 1.5, 40))
    c.n[:] = np.arange(40) % 5
    acc = c.check(c.call(smp))
    assert acc.max() > 0


@pytest.mark.parametrize("V,B", [(32000, 12), (50257, 6), (128256, 6), (151936, 3)])
@pytest.mark.parametrize("draft", [True, False])
def test_chain_vocabularies(smp, V, B, draft):
    rng = np.random.default_rng(V + draft)
    c = Case(rng, B, V, K=3, T=rng.uniform(0.6, 1.2, B), draft=draft)
    c.check(c.call(smp), ok=0.8)


@pytest.mark.parametrize("pad,lead", [(0, 1), (1, 0), (3, 2), (7, 5), (8, 0)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_chain_strides_and_offsets(smp, pad, lead, dt):
    rng = np.random.default_rng(10 * pad + lead)
    c = Case(rng, 24, 777, K=3, pd=dt, qd=dt, pad=pad, lead=lead)
    c.check(c.call(smp))


@pytest.mark.parametrize("mask,cut", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("V,lead", [(40, 0), (1001, 3), (32000, 0)])
def test_chain_masks_and_cutoffs(smp, mask, cut, V, lead):
    rng = np.random.default_rng(V + 2 * mask + cut)
    c = Case(rng, 16, V, K=3, mask=mask, cut=cut, lead=lead)
    if mask:
        # NaN and infinities in masked places are not looked at
        x = c.pr.clone()
        bits = np.unpackbits(c.mask.view(np.uint8), axis=1, bitorder="little")[:, :V].astype(bool)
        hidden = torch.from_numpy(~bits & bits.any(1, keepdims=True)).to(DEV)
        if not cut:
            x[hidden] = torch.where(torch.rand(x.shape, device=DEV) < 0.5, float("nan"), float("inf"))[hidden]
            c.pr.copy_(x)
    c.check(c.call(smp))


def test_mask_of_one_id_and_lowest_values(smp):
    rng = np.random.default_rng(3)
    V = 100
    c = Case(rng, 8, V, K=2)
    c.mask = np.zeros((24, 4), np.uint32)
    for r in range(24):
        j = int(rng.integers(0, V))
        c.mask[r, j >> 5] = 1 << (j & 31)
    c.check(c.call(smp))
    c = Case(rng, 8, V, K=2)
    low = np.finfo(np.float32).min
    for r in range(24):
        c.x[r, rng.choice(V, 90, replace=False)] = low if r % 2 else -np.inf
    c.x[5] = low  # every id alike
    c.pr.copy_(torch.from_numpy(c.x))
    c.check(c.call(smp))


def test_given_drafts_and_draft_temperature_zero(smp):
    rng = np.random.default_rng(5)
    c = Case(rng, 64, 300, K=4, draft=False, sigma=2.0)
    c.tok[:, :] = np.argsort(-c.x.reshape(64, 5, 300)[:, :4], 2)[:, :, 0]
    acc = c.check(c.call(smp))
    assert 0 < acc.mean() < 4
    d = Case(rng, 64, 300, K=4, sigma=2.0)
    d.Tq[:] = 0.0
    d.check(d.call(smp))


def test_greedy_target(smp):
    rng = np.random.default_rng(6)
    B, V = 48, 500
    c = Case(rng, B, V, K=4, T=np.where(np.arange(B) % 2, 0.0, -1.0))
    c.x[:: 7] = np.round(c.x[:: 7])  # ties
    c.pr.copy_(torch.from_numpy(c.x))
    best = c.x.reshape(B, 5, V)[:, :4].argmax(2)
    c.tok[:, :] = np.where(rng.random((B, 4)) < 0.7, best, c.tok)
    out = c.call(smp)
    acc = c.check(out)
    assert acc.max() == 4 and acc.min() == 0
    for b in range(B):
        assert out[2][b, acc[b]] == c.x[b * 5 + acc[b]].argmax() and out[3][b, acc[b]] == 1.0


def test_bad_sequences_and_untouched_rows(smp):
    rng = np.random.default_rng(7)
    B, V, K = 12, 200, 3
    c = Case(rng, B, V, K=K)
    x = c.x.reshape(B, K + 1, V)
    y = c.y.reshape(B, K, V)
    x[0, 0, 5] = np.nan
    x[1, 0, 7] = np.inf
    x[2, 0] = -np.inf
    y[3, 0, 9] = np.nan
    y[4, 0] = -np.inf
    c.tok[5, 0], x[5, 0, :] = -1, x[5, 0, :]  # outside: refused
    x[5, 1] = np.nan  # behind the refusal: not read
    c.tok[6, 0] = V
    c.n[7], c.n[8] = -1, K + 1
    c.T[9], c.Tq[10] = np.nan, np.inf
    c.n[11] = 0
    c.pr.copy_(torch.from_numpy(x.reshape(-1, V)))
    c.qr.copy_(torch.from_numpy(y.reshape(-1, V)))
    acc, path, tok, prob, st = c.call(smp)
    assert st.tolist() == [8, 8, 8, 8, 8, 0, 0, 1, 1, 8, 8, 0]
    for b in (0, 1, 2, 3, 4, 7, 8, 9, 10):
        assert acc[b] == -1 and (tok[b] == -1).all() and (prob[b] == 0).all()
    assert acc[5] == 0 and acc[6] == 0 and acc[11] == 0
    for b in (5, 6, 11):
        r = c.walk(b)
        assert tok[b, 0] == r.tokens[-1]


def test_first_rows_and_no_drafts(smp):
    rng = np.random.default_rng(8)
    B, V, K = 10, 333, 3
    c = Case(rng, B, V, K=K)
    want = c.call(smp)
    # the same sequences with their rows packed in another order
    order = rng.permutation(B)
    c.n[:] = rng.integers(0, K + 1, B)
    want = c.call(smp)
    pf, qf, xs, ys = np.zeros(B, np.int32), np.zeros(B, np.int32), [], []
    for b in order:
        pf[b], qf[b] = len(xs), len(ys)
        xs += list(c.x.reshape(B, K + 1, V)[b, : c.n[b] + 1])
        ys += list(c.y.reshape(B, K, V)[b, : c.n[b]])
    xs, ys = cuda(np.array(xs)), cuda(np.array(ys))
    t, d = rlsampler.DistRows(xs, cuda(c.T), first_row=cuda(pf)), rlsampler.DistRows(ys, cuda(c.Tq), first_row=cuda(qf))
    got = smp.specdec_verify_draft(t, cuda(c.tok), cuda(c.n), cuda(c.u), cuda(c.du), draft=d)
    for g, w in zip(got, (want[0], want[2], None, want[4])):
        assert w is None or np.array_equal(g.cpu().numpy(), w)
    # groups of eight ids start on the row's 16-byte boundaries, and 333 ids
    # leave each row at another one: the same weights, relative to other
    # lanes' maxima and added in another order, so each probability is within
    # EPS of the exact one on both sides
    np.testing.assert_allclose(got[2].cpu().numpy(), want[3], rtol=2 * EPS, atol=0)
    # a block of rows past the end, or before the start
    pf[0], pf[1] = len(xs) - c.n[0], -1
    st = smp.specdec_verify_draft(rlsampler.DistRows(xs, cuda(c.T), first_row=cuda(pf)), cuda(c.tok), cuda(c.n), cuda(c.u), cuda(c.du), draft=d)[3].cpu()
    assert st[0] == 1 and st[1] == 1 and (st[2:] == 0).all()
    # no drafts at all: a plain draw from each row
    z = Case(rng, 6, 200, K=0)
    z.check(z.call(smp))


@pytest.mark.parametrize("T", [1e-6, 1e-3, 50.0, 1e20, 3e38])
def test_extreme_temperatures(smp, T):
    rng = np.random.default_rng(9)
    c = Case(rng, 16, 257, K=2, T=np.full(16, T))
    c.check(c.call(smp), ok=0.9)


def test_uniforms_at_the_ends(smp):
    rng = np.random.default_rng(10)
    c = Case(rng, 16, 400, K=2, sigma=1.0)
    c.u[:8], c.u[8:] = 0.0, np.nextafter(np.float32(1), np.float32(0))
    c.du[::2], c.du[1::2] = 0.0, np.nextafter(np.float32(1), np.float32(0))
    c.check(c.call(smp), ok=0.8)


def test_equal_rows_accept_everything(smp):
    rng = np.random.default_rng(11)
    c = Case(rng, 32, 1000, K=4, noise=0.0)
    c.qr.copy_(c.pr.view(32, 5, 1000)[:, :4].reshape(-1, 1000))
    acc = c.call(smp)[0]
    assert (acc == 4).all()


TREES = {"2": [-1, 0, 0], "3.1": [-1, 0, 0, 0, 1, 2, 3], "4.2.1": [-1] + [0] * 4 + [1, 1, 2, 2, 3, 3, 4, 4] + list(range(5, 13)),
         "line": [-1, 0, 1, 2, 3], "late": [-1, 0, 1, 0, 2, 0, 3], "root": [-1]}


@pytest.mark.parametrize("shape", sorted(TREES))
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("V,pd,lead", [(50, "f32", 0), (1003, "bf16", 1), (4096, "f32", 0)])
def test_tree(smp, shape, draft, V, pd, lead):
    rng = np.random.default_rng(V + len(shape))
    B = 40
    c = Case(rng, B, V, parents=TREES[shape], draft=draft, pd=pd, qd=pd, lead=lead, T=rng.uniform(0.6, 1.2, B), noise=1.0,
             sigma=2.0)
    if not draft:
        for b in range(B):
            for i in range(1, c.N):
                c.tok[b, i] = np.argsort(-c.x[b * c.N + c.parent[b, i]])[rng.integers(0, 4)]  # siblings may repeat
    c.n[::4] = rng.integers(1, c.N + 1, len(c.n[::4]))
    c.T[::6] = 0.0
    c.check(c.call(smp))


def test_tree_masks_cutoffs_and_repeated_siblings(smp):
    rng = np.random.default_rng(21)
    c = Case(rng, 32, 300, parents=TREES["4.2.1"], mask=True, cut=True)
    c.tok[:, 2] = c.tok[:, 1]
    c.tok[:, 4] = 300  # outside
    c.check(c.call(smp))


def test_tree_odd_parents_name_no_node(smp):
    rng = np.random.default_rng(22)
    c = Case(rng, 8, 100, parents=[-1, 0, 0, 1])
    c.parent[:, 2], c.parent[:, 3] = 7, 3  # a later node, and itself
    c.check(c.call(smp))


def test_tree_of_the_most_nodes(smp):
    rng = np.random.default_rng(23)
    c = Case(rng, 2, 64, parents=[-1] + [0] * 255, noise=2.0)
    c.check(c.call(smp))
    d = Case(rng, 2, 64, parents=list(range(-1, 255)), noise=0.0)
    assert d.call(smp)[0].min() >= 0


def test_offsets_past_32_bits(smp):
    """Rows that start beyond 2^31 elements (and 2^32 bytes)."""
    V, R = 151936, 14200
    assert R * V > 2 ** 31
    rng = np.random.default_rng(24)
    c = Case(rng, 1, V, K=1, pd="bf16", qd="bf16")
    big = torch.empty(R, V, dtype=torch.bfloat16, device=DEV)
    big[R - 2:] = c.pr
    f = torch.tensor([R - 2], dtype=torch.int32, device=DEV)
    got = smp.specdec_verify_draft(rlsampler.DistRows(big, cuda(c.T), first_row=f), cuda(c.tok), cuda(c.n), cuda(c.u), cuda(c.du), draft=rlsampler.DistRows(c.qr, cuda(c.Tq)))
    want = c.call(smp)
    assert got[0].cpu().numpy().tolist() == want[0].tolist() and np.array_equal(got[1].cpu().numpy(), want[2])


def test_streams_graphs_and_overlap(smp):
    """Two calls on one handle at once on two streams, and both as replayed graphs, give what each gives alone."""
    rng = np.random.default_rng(25)
    cs = [Case(rng, 20, 8000, K=3), Case(rng, 9, 5000, parents=TREES["3.1"])]
    want = [c.call(smp) for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    args, outs = [], []
    for c in cs:
        t, d = rlsampler.DistRows(c.pr, cuda(c.T)), rlsampler.DistRows(c.qr, cuda(c.Tq))
        args.append((t, d, cuda(c.tok), cuda(c.parent), cuda(c.n), cuda(c.u), cuda(c.du)))

    def go(i):
        t, d, tok, parent, n, u, du = args[i]
        if cs[i].tree:
            return smp.specdec_verify_tree(t, tok, parent, n, u, du, draft=d)
        return smp.specdec_verify_draft(t, tok, n, u, du, draft=d)

    torch.cuda.synchronize()
    for _ in range(3):
        outs = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs.append(go(i))
        torch.cuda.synchronize()
        assert np.array_equal(outs[0][1].cpu().numpy(), want[0][2]) and np.array_equal(outs[1][2].cpu().numpy(), want[1][2])
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs[i] = go(i)
        graphs.append(g)
    for _ in range(3):
        for o in outs[0] + outs[1]:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(outs[0][1].cpu().numpy(), want[0][2]) and np.array_equal(outs[1][2].cpu().numpy(), want[1][2])
    del graphs


def test_first_token_has_the_target_distribution(smp):
    """20,000 sequences over the same pair of rows: the first token that comes
    out is distributed as the target's (5 standard deviations of a share)."""
    rng = np.random.default_rng(26)
    B, V = 20000, 12
    x, y = rng.normal(0, 1.5, V).astype(np.float32), rng.normal(0, 1.5, V).astype(np.float32)
    p, q = ref.dist(x), ref.dist(y)
    pr = torch.from_numpy(x).to(DEV).expand(B * 2, V).contiguous()
    qr = torch.from_numpy(y).to(DEV).expand(B, V).contiguous()
    tok = rng.choice(V, size=(B, 1), p=q).astype(np.int32)
    out = smp.specdec_verify_draft(rlsampler.DistRows(pr), cuda(tok), torch.ones(B, dtype=torch.int32, device=DEV),
                                   cuda(rng.random((B, 1), np.float32)), cuda(rng.random(B, np.float32)), draft=rlsampler.DistRows(qr))
    share = np.bincount(out[1].cpu().numpy()[:, 0], minlength=V) / B
    assert (np.abs(share - p) < 5 * np.sqrt(p * (1 - p) / B) + 1e-4).all()
    assert abs((out[0].float().mean().item()) - np.minimum(p, q).sum()) < 5 * 0.5 / np.sqrt(B)
    # the same with three drawn siblings
    parent = np.tile(np.array([-1, 0, 0, 0], np.int32), (B, 1))
    tok = np.concatenate([np.zeros((B, 1), np.int32), rng.choice(V, size=(B, 3), p=q).astype(np.int32)], 1)
    pr4 = torch.from_numpy(x).to(DEV).expand(B * 4, V).contiguous()
    qr4 = torch.from_numpy(y).to(DEV).expand(B * 4, V).contiguous()
    out = smp.specdec_verify_tree(rlsampler.DistRows(pr4), cuda(tok), cuda(parent), torch.full((B,), 4, dtype=torch.int32, device=DEV),
                                  cuda(rng.random((B, 4), np.float32)), cuda(rng.random(B, np.float32)), draft=rlsampler.DistRows(qr4))
    share = np.bincount(out[2].cpu().numpy()[:, 0], minlength=V) / B
    assert (np.abs(share - p) < 5 * np.sqrt(p * (1 - p) / B) + 1e-4).all()


def test_cutoffs_from_the_sampler(smp):
    """Top-k / top-p through rl_sample_batch_debug's cutoff ids, as a serving
    step has them: every token that comes out lies in the target's kept set."""
    rng = np.random.default_rng(27)
    B, K, V = 8, 3, 32000
    s = rlsampler.Sampler(0, max_batch=B * (K + 1), max_vocab=V, max_history=1)
    c = Case(rng, B, V, K=K)
    prm = lambda R: rlsampler.params_tensor(np.array([(1.0, 0.9, 40, 1.0, 0.0, 0.0)] * R, rlsampler.ROW_PARAMS_DTYPE), DEV)  # noqa: E731
    td = s.sample_debug(c.pr, prm(B * (K + 1)), torch.rand(B * (K + 1), device=DEV))
    dd = s.sample_debug(c.qr, prm(B * K), torch.rand(B * K, device=DEV))
    c.tok = dd[0].view(B, K).cpu().numpy()
    c.cut, c.qcut = td[6][:, 2].cpu().numpy(), dd[6][:, 2].cpu().numpy()
    assert (c.cut >= 0).all() and (c.qcut >= 0).all()
    t = rlsampler.DistRows(c.pr, cuda(c.T), cut=td[6][:, 2])  # a column: stride 3
    d = rlsampler.DistRows(c.qr, cuda(c.Tq), cut=dd[6][:, 2])
    got = smp.specdec_verify_draft(t, cuda(c.tok), cuda(c.n), cuda(c.u), cuda(c.du), draft=d)
    want = c.call(smp)
    assert np.array_equal(got[1].cpu().numpy(), want[2])
    c.check(want)
    s.close()


@pytest.mark.parametrize("pad,first", [("given", 600), ("drawn", 600), ("given", 5000), ("drawn", 5000)])
def test_first_ids_at_the_edge_of_the_weights(smp, pad, first):
    """A draw with u = 0 where the row's first ids weigh about 2^-126 of its
    largest, in steps around that: whatever counts there, the token is an id of
    the row and none before it has any weight by its own."""
    B, V = 400, 20000
    rng = np.random.default_rng(40)
    m = rng.choice([0.0, 3.3, -7.1, 400.7, -9000.3], B)
    x = np.full((B, V), -np.inf, np.float32)
    x[:, V - 5] = m
    gap = (126.0 + np.linspace(-1.5, 1.5, B)) * np.log(2.0)
    x[:, :first] = (x[:, V - 5].astype(np.float64) - gap)[:, None]
    rows = torch.from_numpy(x).to(DEV)
    zero = torch.zeros(B, device=DEV)
    n = torch.zeros(B, dtype=torch.int32, device=DEV)
    none = torch.empty(B, 0, dtype=torch.int32, device=DEV)
    kw = {}
    if pad == "drawn":  # one draft that the target refuses: the token comes from max(p - q, 0)
        n += 1
        none = torch.full((B, 1), V - 3, dtype=torch.int32, device=DEV)
        q = torch.full((B, V), -np.inf, device=DEV)
        q[:, V - 3] = 1.0
        kw["draft"] = rlsampler.DistRows(q)
        rows = rows.repeat_interleave(2, 0).contiguous()
    acc, tok, prob, st = smp.specdec_verify_draft(rlsampler.DistRows(rows), none, n, torch.zeros(none.shape, device=DEV), zero, **kw)
    tok = tok[:, 0].cpu().numpy()
    assert (st == 0).all() and (acc == 0).all()
    assert np.isin(tok, [0, V - 5]).all(), tok[~np.isin(tok, [0, V - 5])]
    assert (tok[gap < 124.5 * np.log(2.0)] == 0).all()


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("drawn", [False, True])
def test_products_beyond_the_range_of_floats(smp, sign, drawn):
    """At a temperature of 1e-38 logits times 1 / T leave the range of floats:
    all of a row's probability is on its largest logit, wherever that lies."""
    V, places = 128256, [0, 3, 700, 1100, 1537, 64000, 128255]
    B = len(places)
    rng = np.random.default_rng(41)
    x = (rng.random((B, V)) * 8 + (10 if sign > 0 else -40)).astype(np.float32)
    for b, j in enumerate(places):
        x[b, j] = 19.0 if sign > 0 else -5.0
    T = torch.full((B,), 1e-38, device=DEV)
    rows = torch.from_numpy(x).to(DEV)
    du = torch.tensor([0.0, 0.3, 0.6, 0.9, 0.99, 0.5, 0.1], device=DEV)
    K = 1 if drawn else 0
    drafts = torch.tensor([[(j + 1) % V] for j in places], dtype=torch.int32, device=DEV)[:, :K].contiguous()
    kw = {}
    if drawn:
        y = x.copy()
        y[np.arange(B), [(j + 1) % V for j in places]] = 20.0
        kw["draft"] = rlsampler.DistRows(torch.from_numpy(y).to(DEV), T)
        rows = rows.repeat_interleave(2, 0).contiguous()
    acc, tok, prob, st = smp.specdec_verify_draft(rlsampler.DistRows(rows, T), drafts, torch.full((B,), K, dtype=torch.int32, device=DEV),
                                                  torch.full((B, K), 0.5, device=DEV), du, **kw)
    assert (st == 0).all() and (acc == 0).all()
    assert tok[:, 0].tolist() == places and (prob[:, 0] == 1).all()


@pytest.mark.parametrize("T", [1e-4, 1e-6, 1e-7, 1e-8, 1e-9, 1e-12, 1e-20, 1e-30, 1e-37, 2e-38])
@pytest.mark.parametrize("shift", [-40.0, -3.0, 0.0, 12.0, 900.0])
def test_small_temperatures_at_any_level(smp, T, shift):
    """Logits over T far above 1, where products lose the fractions that decide:
    a few ids lie within a few T of the largest (as far as f32 can tell them
    apart), the others below."""
    B, V = 12, 9000
    rng = np.random.default_rng(43)
    c = Case(rng, B, V, K=2, T=np.full(B, T), sigma=2.0)
    step = np.abs(np.spacing(np.float32(abs(shift) + 8)))
    for rows in (c.pr, c.qr):
        x = rows.cpu().numpy() * np.float32(0.5)
        x = np.minimum(x, 6.0).astype(np.float32)
        for r in range(len(x)):
            near = rng.choice(V, 6, replace=False)
            x[r, near] = 8.0 - np.round(rng.random(6) * 5) * max(step, np.float32(T))
        rows.copy_(torch.from_numpy((x.astype(np.float64) + shift).astype(np.float32)))
    c.x, c.y = c.pr.cpu().numpy(), c.qr.cpu().numpy()
    c.tok[:] = np.argmax(c.x.reshape(B, 3, V)[:, :2], 2).reshape(c.tok.shape)
    c.check(c.call(smp), ok=0.9)
