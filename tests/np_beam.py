"""Beam search in 64 bits, one candidate at a time: the definition that the GPU tests hold the kernels against."""
import numpy as np


def penalised(z, history, repetition=0.0, frequency=0.0, presence=0.0):
    """fp32 row after the penalties over a list of ids, three rounded operations as born_sample's."""
    z = z.astype(np.float32).copy()
    v = len(z)
    ids, counts = np.unique([t for t in history if 0 <= t < v], return_counts=True)
    for t, c in zip(ids.astype(int), counts):
        if repetition not in (0.0, 1.0):
            z[t] = z[t] / np.float32(repetition) if z[t] > 0 else z[t] * np.float32(repetition)
        if frequency or presence:
            z[t] = z[t] - (np.float32(frequency) * np.float32(c) + np.float32(presence))
    return z


OK, ALL_MASKED, NAN, POS_INF, FINISHED, DEAD = 0, 1, 2, 3, 6, 8


def row_values(z, score, temperature):
    """(status, values of all tokens in 64 bits or None)."""
    if np.isnan(score):
        return NAN, None
    if score == np.inf:
        return POS_INF, None
    if score == -np.inf:
        return DEAD, None
    if np.isnan(z).any():
        return NAN, None
    if (z == np.inf).any():
        return POS_INF, None
    if (z == -np.inf).all():
        return ALL_MASKED, None
    t = np.float64(np.float32(temperature if temperature else 1.0))
    x = z.astype(np.float64)
    top = x.max()
    with np.errstate(over="ignore"):
        lse = np.log(np.exp((x - top) / t).sum())
    return OK, np.float64(np.float32(score)) + (x - top) / t - lse


def step(rows, scores, stops=(), temperature=0.0, keep_slots=False):
    """One group: rows [K] of fp32 logits with penalties and mask applied (-inf).  Returns a dict."""
    K, V = len(rows), len(rows[0])
    status, cand, ended = [], [], []
    for b in range(K):
        s, v = row_values(rows[b], scores[b], temperature)
        status.append(s)
        if v is None:
            continue
        order = np.argsort(-v, kind="stable")[:K + len(stops)]
        cand += [(-v[t], b, int(t)) for t in order if v[t] > -np.inf]
        cand += [(-v[t], b, int(t)) for t in set(stops) if 0 <= t < V and v[t] > -np.inf and t not in order]
    cand.sort()
    ended = [c for c in cand[:K] if c[2] in stops]
    going = [c for c in cand if c[2] not in stops][:K]
    place = [None] * K
    if keep_slots:
        late = []
        for c in going:
            if place[c[1]] is None:
                place[c[1]] = c
            else:
                late.append(c)
        for r in range(K):
            if place[r] is None and late:
                place[r] = late.pop(0)
    else:
        place[:len(going)] = going
    place = [c if c else (np.inf, r, -1) for r, c in enumerate(place)]
    ended = ended + [(np.inf, -1, -1)] * (K - len(ended))
    return dict(parent=[c[1] for c in place], token=[c[2] for c in place], score=[-c[0] for c in place], status=status,
                end_parent=[c[1] for c in ended], end_token=[c[2] for c in ended], end_score=[-c[0] for c in ended],
                best=-going[0][0] if going else -np.inf)


class Pool:
    """The best K ended hypotheses of one group: (score, step, parent, token), best first."""

    def __init__(self, beams):
        self.beams, self.items, self.done = beams, [], False

    def add(self, out, step_no, length_penalty, early_stop):
        norm = np.float64(step_no + 1) ** np.float64(np.float32(length_penalty))
        for p, t, s in zip(out["end_parent"], out["end_token"], out["end_score"]):
            if t < 0:
                break
            v = np.float32(s / norm)
            if len(self.items) == self.beams and not v > self.items[-1][0]:
                continue
            at = len(self.items)
            while at > 0 and v > self.items[at - 1][0]:
                at -= 1
            self.items.insert(at, (v, step_no, p, t))
            del self.items[self.beams:]
        full = len(self.items) == self.beams
        if out["best"] == -np.inf or (full and (early_stop or not np.float32(out["best"] / norm) > self.items[-1][0])):
            self.done = True
