"""Plain 64-bit restatement of the verification of drafted tokens
(rl_specdec_verify_draft, rl_specdec_verify_tree), numpy only.

walk() goes through one sequence and says how near each decision was to its
border, so that a comparison can tell a wrong token from one that lies within
the rounding of f32 weights of the right one.
"""
import numpy as np


def dist(x, T=1.0, mask=None, cut=None):
    """Probabilities of one row, or None where it has none (NaN or +inf in a
    kept place, no id left, T not finite)."""
    x = np.asarray(x, np.float64).copy()
    V = len(x)
    if not np.isfinite(T):
        return None
    keep = np.ones(V, bool)
    if mask is not None:
        bits = np.unpackbits(np.ascontiguousarray(mask).view(np.uint8), bitorder="little")[:V].astype(bool)
        if bits.any():
            keep = bits
    if cut is not None and 0 <= cut < V:
        ids = np.arange(V)
        keep &= ~((x < x[cut]) | ((x == x[cut]) & (ids > cut)))
    x[~keep] = -np.inf
    if np.isnan(x).any() or (x == np.inf).any() or not (x > -np.inf).any():
        return None
    if T <= 0:
        p = np.zeros(V)
        p[int(np.argmax(x))] = 1.0  # the first of equal maxima
        return p
    e = np.exp((x - x.max()) / T)
    e[e < 2.0 ** -126] = 0.0
    return e / e.sum()


class Walk:
    """What walk() found: accepted nodes and tokens, the drawn token, their
    target probabilities, the smallest distance of an accept test from its
    border (relative to the terms of the test), and the running sums next to
    the draw's target."""

    def __init__(self):
        self.path, self.tokens, self.probs = [], [], []
        self.bad = False
        self.accept_margin = np.inf
        self.run = self.target = self.w = None


def walk(p_of, q_of, children, token, u_of, draw_u, greedy=False):
    """p_of(node), q_of(node): rows of probabilities (None: the walk fails, or
    for q_of that the children were given)."""
    r = Walk()
    node = 0
    while True:
        p = p_of(node)
        kids = children(node)
        q = q_of(node) if kids and not greedy else None
        if p is None or (isinstance(q, str) and q == "bad"):
            r.bad = True
            return r
        w, went, C = p.copy(), False, 0.0
        for c in kids:
            x = token(c)
            inside = 0 <= x < len(p)
            wx = w[x] if inside else 0.0
            qx = (q[x] if inside else 0.0) if q is not None else (1.0 if inside else 0.0)
            if greedy:
                yes = wx > 0.0
            else:
                lhs = float(u_of(c)) * qx * w.sum()
                yes = lhs < wx
                # against the terms that the test is computed from
                px = p[x] if inside else 0.0
                terms = lhs + px + (C * qx if q is not None else 0.0)
                exactly = C * qx if q is not None else px - wx
                r.accept_margin = min(r.accept_margin, abs(lhs - (px - exactly)) / terms if terms > 0 else np.inf)
            if yes:
                r.path.append(c)
                r.tokens.append(x)
                r.probs.append(p[x])
                node, went = c, True
                break
            if q is not None:
                C += w.sum()
                w = np.maximum(w - w.sum() * q, 0.0)
            elif inside and not greedy:
                w[x] = 0.0
        if went:
            continue
        if greedy:
            w = p
        if not w.sum() > 0:
            w = p.copy()
        r.w, r.run = w, np.cumsum(w)
        r.target = float(draw_u) * r.run[-1]
        hit = np.flatnonzero(r.run > r.target)
        x = int(hit[0]) if len(hit) else int(np.flatnonzero(w > 0)[-1])
        r.tokens.append(x)
        r.probs.append(p[x])
        r.p = p
        return r
