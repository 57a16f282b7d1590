"""sample_logits in 64 bits, and a dispatch of it."""
from __future__ import annotations

import numpy as np

from linear_cases import Rows, dispatch

NONE = 0xFFFFFFFF


def order_of(row):
    """Indices of what can be kept, largest first, equal ones by index."""
    live = np.flatnonzero(row > -np.inf)  # neither NaN nor -infinity
    return live[np.lexsort((live, -row[live]))]


def distribution(row, temperature, k, p, min_p):
    """Indices kept, ascending, and their probabilities."""
    order = order_of(row)
    if len(order) == 0:
        return order, np.zeros(0)
    if not temperature > 0:
        return order[:1], np.ones(1)
    x = row[order].astype(np.float64)
    if np.isinf(x[0]):
        w = (x == x[0]).astype(np.float64)
    else:
        w = np.exp((x - x[0]) / float(temperature))
    n = len(order) if k == 0 else min(int(k), len(order))
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[:n])[:-1]])
        n = max(1, int((before < max(float(p), 0.0) * w[:n].sum()).sum()))
    keep = np.ones(n, bool)
    if min_p > 0:
        keep = (w[:n] >= float(min_p)) | (x[:n] == x[0])
    kept, w = order[:n][keep], w[:n][keep]
    at = np.argsort(kept)
    return kept[at], w[at] / w.sum()


class Sample:
    def __init__(self, logits, temperature=1.0, k=0, p=1.0, min_p=0.0, u=None, seed=0):
        self.logits = np.asarray(logits, np.float32)
        n = len(self.logits)
        self.temperature, self.p, self.min_p = (np.broadcast_to(np.asarray(v, np.float32), n).copy()
                                                for v in (temperature, p, min_p))
        self.k = np.broadcast_to(np.asarray(k, np.uint32), n).copy()
        rng = np.random.default_rng(seed)
        self.u = rng.random(n, np.float32) if u is None else np.broadcast_to(np.asarray(u, np.float32), n).copy()

    def run(self, gpu, pad=0, shift=0, static=False):
        n, vocab = self.logits.shape
        x = Rows(gpu, self.logits, pad, shift)
        up = gpu.upload_bytes
        tokens, probs = up(np.full(n + 2, 7, np.uint32)), gpu.upload_f32(np.full(n + 2, 7, np.float32))
        dispatch(gpu, "sample_logits", [x.buffer, up(self.temperature), up(self.k), up(self.p), up(self.min_p), up(self.u),
                                        tokens, probs], [n, vocab, x.stride], [x.offset, 0, 0, 0, 0, 0, 4, 4], static)
        tokens, probs = tokens.read(np.uint32, n + 2), probs.read(np.float32, n + 2)
        assert tokens[0] == tokens[-1] == 7 and probs[0] == probs[-1] == 7
        return tokens[1:-1], probs[1:-1]

    def check(self, gpu, **how):
        """Equal tokens, unless the number stands within 1e-10 of a border (as
        far as weights in 2^-45 and sums in 64 bits can move it)."""
        tokens, probs = self.run(gpu, **how)
        for r, row in enumerate(self.logits):
            kept, share = distribution(row, self.temperature[r], self.k[r], self.p[r], self.min_p[r])
            if len(kept) == 0:
                assert tokens[r] == NONE and probs[r] == 0, r
                continue
            up_to = np.cumsum(share)
            u = min(max(float(self.u[r]), 0.0), 1.0) if self.u[r] == self.u[r] else 0.0
            at = min(int(np.searchsorted(up_to, u * up_to[-1], side="right")), len(kept) - 1)
            while share[at] == 0:
                at -= 1
            assert tokens[r] == kept[at] or np.abs(up_to - u).min() < 1e-10, (r, tokens[r], kept[at])
            where = np.searchsorted(kept, tokens[r])
            # Rounded once, and from weights off by 2^-45 of the largest.
            assert abs(probs[r] - share[where]) <= 1.01 * 2.0 ** -24 * share[where] + 2.0 ** -36, r
        return tokens, probs
