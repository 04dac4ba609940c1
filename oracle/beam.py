"""Beam selection, the beams' loop control and their reordering, written from
the definitions in numpy and 64 bits (include/pesti_sampler.h); the checker of
the beam search tests."""
import numpy as np

NEG = -np.inf


def row_logp(x):
    """(logp [V], log sum exp) of one row in 64 bits.  NaN counts as -inf; the
    +inf entries of a row share its probability."""
    x = np.where(np.isnan(x), NEG, x).astype(np.float64)
    m = x.max()
    if m == NEG:
        return np.full(x.shape, NEG), NEG
    if m == np.inf:
        n = np.count_nonzero(x == np.inf)
        return np.where(x == np.inf, -np.log(n), NEG), np.inf
    s = np.exp(x - m).sum()
    with np.errstate(invalid="ignore"):
        return (x - m) - np.log(s), m + np.log(s)


def select(x, W, K, cum=None, done=None):
    """x [G*W, V] (the logits' values as f32/f64) -> score [G, K] f64, token, parent, lse [G*W]."""
    rows, V = x.shape
    G = rows // W
    score = np.full((G, K), NEG)
    token, parent = np.full((G, K), -1, np.int32), np.full((G, K), -1, np.int32)
    lse = np.full(rows, NEG)
    for g in range(G):
        if done is not None and done[g]:
            continue
        have = []
        for w in range(W):
            row = x[g * W + w]
            logp, lse[g * W + w] = row_logp(row)
            c = 0.0 if cum is None else float(cum[g, w])
            if not c > NEG:
                continue
            row = np.where(np.isnan(row), NEG, row).astype(np.float64)
            order = np.lexsort((np.arange(V), -row))[:K]
            for r, v in enumerate(order):
                if row[v] > NEG and logp[v] > NEG:
                    have.append((-(c + logp[v]), w, r, int(v)))
        have.sort()
        for r, (neg, w, _, v) in enumerate(have[:K]):
            score[g, r], token[g, r], parent[g, r] = -neg, v, w
    return score, token, parent, lse


class Beams:
    """One group's loop control (pesti_beam_advance)."""

    def __init__(self, W, max_tokens, max_seq_len, stop=(), length_penalty=1.0, early_stop=False):
        self.W, self.max_tokens, self.max_seq_len = W, max_tokens, max_seq_len
        self.limit, self.stop, self.alpha, self.early = min(max_tokens, max_seq_len), set(stop), length_penalty, early_stop
        self.cum = [0.0] + [NEG] * (W - 1)
        self.last, self.parent = [0] * W, [-1] * W
        # rows of `limit` places, as the device holds them: a dead beam's row stays as it was, so a
        # candidate that names one continues whatever the first `count` places hold
        self.hist = [[0] * self.limit for _ in range(W)]
        self.pool, self.count, self.done = [], 0, 0

    def _finish(self, s, tokens):
        norm = np.float32(s)
        if len(self.pool) < self.W:
            self.pool.append((norm, tokens))
            return
        low = min(range(self.W), key=lambda i: (self.pool[i][0], -i))
        if norm > self.pool[low][0]:
            self.pool[low] = (norm, tokens)

    def advance(self, score, token, parent):
        W = self.W
        self.parent = [-1] * W
        if self.done:
            return
        if self.count >= self.limit:
            self.done = 3 if self.count >= self.max_seq_len else 2
            return
        live = []
        for r, (s, t, p) in enumerate(zip(score, token, parent)):
            if t < 0 or not 0 <= p < W:
                continue
            if int(t) in self.stop:
                if r < W:
                    self._finish(float(s) / (self.count + 1) ** self.alpha, self.hist[p][:self.count])
            elif len(live) < W:
                live.append((float(s), int(t), int(p)))
        c = self.count
        new = [self.hist[p][:c] + [t] + self.hist[w][c + 1:] for w, (_, t, p) in enumerate(live)]
        self.hist = new + self.hist[len(new):]
        for w in range(W):
            self.cum[w] = live[w][0] if w < len(live) else NEG
            if w < len(live):
                self.last[w], self.parent[w] = live[w][1], live[w][2]
        self.count += 1
        if self.count >= self.limit:
            for w in range(len(live)):
                self._finish(self.cum[w] / self.count ** self.alpha, self.hist[w][:self.count])
            self.done = 3 if self.count >= self.max_seq_len else 2
        elif not live:
            self.done = 1
        elif len(self.pool) >= W:
            best = max(self.cum)
            ahead = max(best / (self.count + 1) ** self.alpha, best / float(self.limit) ** self.alpha)
            if self.early or min(p[0] for p in self.pool) >= ahead:
                self.done = 1
