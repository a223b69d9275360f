"""The work of beam-search decoding that a program hands to this library, as timed cases.

An *op* is one call of the decode loop, in the order in which the loop makes them:

  linear     the output head: logits = act(hidden x weight^T + bias) + residual
  step       one step of the search: scores, stop tokens and the best beams of every group
  reorder    the states (attention caches, recurrent states) follow the beams that go on, in place
  sequences  the token sequences read out of the tables that the steps left

Vocabularies, batches and histories are those of the benchmark configurations and of the tests; hidden
sizes and cache layouts are generic.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}

_STEP = dict(op="step", groups=1, beams=4, vocab=32000, dtype="f32", mask=False, history=0, stops=1, temperature=1.0,
             repetition=1.0, frequency=0.0, presence=0.0, keep_slots=True, first=False)
_REORDER = dict(op="reorder", groups=1, beams=4, buffers=1, planes=1, positions=1, width=64, dtype="bf16", ragged=False)
_SEQUENCES = dict(op="sequences", groups=1, beams=4, steps=64)
_LINEAR = dict(op="linear", rows=1, hidden=2048, vocab=32000, out="f32", bias=False, residual=False, activation="none",
               scale=1.0)


def listed():
    return [
        # one user, one token: the smallest step, all latency
        {**_STEP, "name": "step_one", "vocab": 32000},
        # a few users, odd vocabulary, a repetition penalty over the text so far
        {**_STEP, "name": "step_ragged", "groups": 9, "beams": 5, "vocab": 50257, "dtype": "bf16", "history": 200,
         "repetition": 1.2, "keep_slots": False},
        # a grammar's mask lets one token in twenty through
        {**_STEP, "name": "step_constrained", "groups": 32, "beams": 8, "vocab": 151936, "dtype": "bf16", "mask": True,
         "stops": 2},
        # a full batch: 256 rows in groups of four, penalties over 512 tokens
        {**_STEP, "name": "step_b64", "groups": 64, "beams": 4, "vocab": 128256, "history": 512, "temperature": 0.7,
         "frequency": 0.5, "presence": 0.3},
        # one user's attention cache after a short prompt
        {**_REORDER, "name": "reorder_one", "buffers": 16, "planes": 8, "positions": 256, "width": 128, "ragged": True},
        # recurrent states of odd width, rows at any alignment
        {**_REORDER, "name": "reorder_odd", "groups": 7, "beams": 6, "buffers": 3, "width": 40961, "dtype": "f32"},
        # the attention caches of a batch, sequences of different lengths
        {**_REORDER, "name": "reorder_b32", "groups": 32, "beams": 4, "buffers": 16, "planes": 8, "positions": 1024,
         "width": 64, "ragged": True},
        # a short answer of one user
        {**_SEQUENCES, "name": "sequences_one", "steps": 64},
        # long answers of a batch
        {**_SEQUENCES, "name": "sequences_b64", "groups": 64, "beams": 8, "steps": 4096},
        # one row: the head is as fast as its weights are read
        {**_LINEAR, "name": "linear_one", "rows": 1, "hidden": 2048, "vocab": 32000, "out": "bf16"},
        # a few rows, odd sizes, scores of another model added to the logits
        {**_LINEAR, "name": "linear_ragged", "rows": 37, "hidden": 1000, "vocab": 50257, "bias": True, "residual": True},
        # a full batch with capped logits
        {**_LINEAR, "name": "linear_b256", "rows": 256, "hidden": 4096, "vocab": 128256, "activation": "tanh",
         "scale": 30.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _draw_vocab(rng, lo, hi):
    """Log-uniform; two in three a multiple of 64, as vocabularies are padded to, the others as they fall."""
    v = _log_int(rng, lo, max(lo, hi))
    return v if rng.random() < 0.34 else max(64, v // 64 * 64)


def draw(rng):
    op = rng.choice(["step", "step", "reorder", "sequences", "linear"])
    if op == "step":
        beams = rng.randint(1, 16)
        groups = _log_int(rng, 1, 256 // beams)
        vocab = _draw_vocab(rng, 1000, min(262144, 33_000_000 // (groups * beams)))
        history = _log_int(rng, 1, 1024) if rng.random() < 0.5 else 0
        kind = rng.choice(["repetition", "counts"]) if history else ""
        return {**_STEP, "groups": groups, "beams": beams, "vocab": vocab, "dtype": rng.choice(["f32", "bf16"]),
                "mask": rng.random() < 0.3, "history": history, "stops": rng.randint(0, 3),
                "temperature": rng.choice([1.0, round(rng.uniform(0.5, 1.5), 3)]),
                "repetition": 1.2 if kind == "repetition" else 1.0, "frequency": 0.5 if kind == "counts" else 0.0,
                "presence": 0.3 if kind == "counts" else 0.0, "keep_slots": rng.random() < 0.5,
                "first": rng.random() < 0.15}
    if op == "reorder":
        beams = rng.randint(2, 16)
        groups = _log_int(rng, 1, 32)
        if rng.random() < 0.3:
            return {**_REORDER, "groups": groups, "beams": beams, "buffers": rng.randint(1, 8),
                    "width": _log_int(rng, 16, 100000), "dtype": rng.choice(["f32", "bf16"])}
        width = rng.choice([64, 80, 128])
        planes = rng.choice([1, 4, 8])
        buffers = rng.choice([2, 8, 16, 32])
        most = 1_000_000_000 // (groups * beams * width * planes * buffers)
        return {**_REORDER, "groups": groups, "beams": beams, "buffers": buffers, "planes": planes, "width": width,
                "positions": _log_int(rng, 1, max(1, min(4096, most))), "dtype": rng.choice(["f32", "bf16"]),
                "ragged": rng.random() < 0.8}
    if op == "sequences":
        return {**_SEQUENCES, "groups": _log_int(rng, 1, 64), "beams": rng.randint(1, 8), "steps": _log_int(rng, 1, 4096)}
    hidden = 8 * _log_int(rng, 16, 1024)
    vocab = _draw_vocab(rng, 256, min(262144, 520_000_000 // hidden))
    rows = _log_int(rng, 1, min(512, max(1, 256 * 4096 * 128256 // (hidden * vocab))))
    activation = rng.choice(["none", "none", "relu", "sigmoid", "tanh", "gelu", "silu"])
    return {**_LINEAR, "rows": rows, "hidden": hidden, "vocab": vocab, "out": rng.choice(["f32", "bf16"]),
            "bias": rng.random() < 0.5, "residual": rng.random() < 0.4, "activation": activation,
            "scale": 30.0 if activation == "tanh" else 1.0}


# ---- inputs -----------------------------------------------------------------------------
def _words(bits):
    weight = 2 ** torch.arange(32, device="cuda", dtype=torch.int64)
    word = (bits.view(bits.shape[0], -1, 32) * weight).sum(-1)
    return torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)


def _prepare_step(case, g):
    N, K, V = case["groups"], case["beams"], case["vocab"]
    R = N * K
    state = {}
    z = torch.randn((R, V), generator=g, device="cuda") * 2.0
    likely = torch.randint(0, V, (R, 12), generator=g, device="cuda")  # a few tokens that the model expects
    z.scatter_add_(1, likely, 4.0 + 4.0 * torch.rand((R, 12), generator=g, device="cuda"))
    stops = torch.randperm(V, generator=g, device="cuda")[:case["stops"]]
    # the end of the text is likely for some beams
    z[:, stops] += 9.0 * (torch.rand((R, case["stops"]), generator=g, device="cuda") < 0.3)
    state["logits"] = z.to(_DTYPES[case["dtype"]])
    if case["first"]:
        scores = torch.full((N, K), -math.inf, device="cuda")
        scores[:, 0] = 0.0
    else:
        scores = -20.0 - 2.0 * torch.rand((N, K), generator=g, device="cuda").sort(dim=1).values
    state["scores"] = scores.view(R)
    state["stops"] = sorted(stops.tolist())
    if case["mask"]:
        bits = torch.rand((R, (V + 31) // 32 * 32), generator=g, device="cuda") < 0.05
        bits[:, V:] = False
        bits[:, 0] |= ~bits.any(dim=1)
        state["mask"] = _words(bits)
    if case["history"]:
        state["history"] = torch.randint(0, V, (R, case["history"]), generator=g, device="cuda", dtype=torch.int32)
    return state


def _surviving(N, K, g):
    """Parents as a step leaves them: a beam that goes on keeps its row, the rows of the others are taken over."""
    parent = torch.randint(0, K, (N, K), generator=g, device="cuda")
    slot = torch.arange(K, device="cuda").expand(N, K)
    alive = torch.zeros((N, K), dtype=torch.bool, device="cuda").scatter_(1, parent, True)
    return torch.where(alive, slot, parent).to(torch.int32).view(-1)


def _prepare_reorder(case, g):
    N, K = case["groups"], case["beams"]
    shape = (case["buffers"], N * K, case["planes"], case["positions"], case["width"])
    state = {"buffers": torch.randn(shape, generator=g, device="cuda", dtype=_DTYPES[case["dtype"]]),
             "parents": _surviving(N, K, g)}
    if case["ragged"]:
        state["lens"] = torch.randint(0, case["positions"] + 1, (N,), generator=g, device="cuda", dtype=torch.int32)
    return state


def _prepare_sequences(case, g):
    N, K, T = case["groups"], case["beams"], case["steps"]
    tokens = torch.randint(0, 128256, (T, N * K), generator=g, device="cuda", dtype=torch.int32)
    parents = torch.randint(0, K, (T, N, K), generator=g, device="cuda", dtype=torch.int32).view(T, N * K)
    # hypotheses that ended at some step, and one place in eight of the list still free
    end = torch.randint(0, T, (N, K), generator=g, device="cuda", dtype=torch.int32)
    end = torch.where(torch.rand((N, K), generator=g, device="cuda") < 0.125, torch.full_like(end, -1), end)
    return {"tokens": tokens, "parents": parents, "end_step": end,
            "end_parent": torch.randint(0, K, (N, K), generator=g, device="cuda", dtype=torch.int32),
            "end_token": torch.randint(0, 128256, (N, K), generator=g, device="cuda", dtype=torch.int32)}


def _prepare_linear(case, g):
    M, H, V, out = case["rows"], case["hidden"], case["vocab"], _DTYPES[case["out"]]
    state = {"x": torch.randn((M, H), generator=g, device="cuda").to(torch.bfloat16),
             "weight": torch.randn((V, H), generator=g, device="cuda", dtype=torch.bfloat16) * (2.5 / math.sqrt(H))}
    if case["bias"]:
        state["bias"] = torch.randn((V,), generator=g, device="cuda")
    if case["residual"]:
        state["residual"] = torch.randn((M, V), generator=g, device="cuda").to(out)
    return state


_PREPARE = {"step": _prepare_step, "reorder": _prepare_reorder, "sequences": _prepare_sequences, "linear": _prepare_linear}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"case": case, **_PREPARE[case["op"]](case, g)}


# ---- the plain forms ----------------------------------------------------------------------
def _penalised(case, z, state):
    """Penalties over the history, then the mask: born_sample's order, three 32-bit roundings."""
    if "history" in state:
        ids = state["history"].long()
        count = torch.zeros_like(z).scatter_add_(1, ids, torch.ones_like(ids, dtype=torch.float32))
        if case["repetition"] != 1.0:
            r = torch.tensor(case["repetition"], dtype=torch.float32, device="cuda")
            z = torch.where(count > 0, torch.where(z > 0, z / r, z * r), z)
        if case["frequency"] or case["presence"]:
            f = torch.tensor(case["frequency"], dtype=torch.float32, device="cuda")
            p = torch.tensor(case["presence"], dtype=torch.float32, device="cuda")
            z = torch.where(count > 0, z - (f * count + p), z)
    if "mask" in state:
        t = torch.arange(z.shape[1], device="cuda")
        bit = (state["mask"][:, t >> 5] >> (t & 31).to(torch.int32)) & 1
        z = torch.where(bit != 0, z, -math.inf)
    return z


def _in_slots(parent, token, score, K):
    """The best child of a beam takes the beam's own row, the other children the rows that are left."""
    N = parent.shape[0]
    lives = token >= 0
    same = (parent[:, :, None] == parent[:, None, :]) & lives[:, None, :]
    earlier = torch.ones((K, K), dtype=torch.bool, device="cuda").tril(-1)
    stays = lives & ~(same & earlier).any(-1)
    taken = torch.zeros((N, K + 1), dtype=torch.bool, device="cuda")
    taken = taken.scatter(1, torch.where(stays, parent, K), True)[:, :K]
    free = torch.sort(taken.to(torch.int8), dim=1, stable=True).indices  # free rows first, ascending
    nth = torch.cumsum((~stays).long(), 1) - 1
    slot = torch.where(stays, parent, free.gather(1, nth.clamp(min=0)))
    parent = torch.where(lives, parent, slot)
    back = torch.empty_like(slot).scatter_(1, slot, torch.arange(K, device="cuda").expand(N, K))
    return parent.gather(1, back), token.gather(1, back), score.gather(1, back)


def _plain_step(state):
    case = state["case"]
    N, K, V = case["groups"], case["beams"], case["vocab"]
    z = _penalised(case, state["logits"].float(), state)
    # ranked in 64 bits: candidates of different beams come as near to each other as they like
    x = z.double() / float(torch.tensor(case["temperature"], dtype=torch.float32))
    top = x.amax(1, keepdim=True)
    logp = x - top - torch.log(torch.exp(x - top).sum(1, keepdim=True))
    total = (state["scores"].double()[:, None] + logp).view(N, K * V)
    stop = torch.zeros(V, dtype=torch.bool, device="cuda")
    stop[torch.tensor(state["stops"], dtype=torch.int64, device="cuda")] = True
    # more than can be needed, in index order, then by value: equal values stay in index order
    best = torch.topk(total, min(K * V, K + K * len(state["stops"]) + 64), dim=1).indices.sort(dim=1).values
    value, order = torch.sort(total.gather(1, best), dim=1, descending=True, stable=True)
    best = best.gather(1, order)
    beam, token = best // V, best % V
    ends = stop[token]
    # the first K that are no stop tokens go on
    _, at = torch.sort(ends.to(torch.int8), dim=1, stable=True)
    at = at[:, :K]
    score = torch.where(ends.gather(1, at), -math.inf, value.gather(1, at))
    dead = score == -math.inf
    parent = torch.where(dead, torch.arange(K, device="cuda").expand(N, K), beam.gather(1, at))
    nxt = torch.where(dead, -1, token.gather(1, at))
    if case["keep_slots"]:
        parent, nxt, score = _in_slots(parent, nxt, score, K)
    out = {"parent": parent.reshape(-1).int(), "token": nxt.reshape(-1).int(), "score": score.reshape(-1).float()}
    if state["stops"]:
        # the stop tokens among the K best of all end here
        ended = ends[:, :K] & (value[:, :K] > -math.inf)
        _, at = torch.sort((~ended).to(torch.int8), dim=1, stable=True)
        ended = ended.gather(1, at)
        out["end_parent"] = torch.where(ended, beam.gather(1, at), -1).int()
        out["end_token"] = torch.where(ended, token.gather(1, at), -1).int()
        out["end_score"] = torch.where(ended, value.gather(1, at), -math.inf).float()
    return out


def _plain_reorder(state):
    case, buffers = state["case"], state["buffers"]
    N, K, P = case["groups"], case["beams"], case["positions"]
    source = state["parents"].long() + torch.arange(N, device="cuda").repeat_interleave(K) * K
    moved = buffers[:, source]
    if "lens" in state:
        used = torch.arange(P, device="cuda") < state["lens"].repeat_interleave(K)[:, None]
        moved = torch.where(used[None, :, None, :, None], moved, buffers)
    buffers.copy_(moved)
    return buffers


def _plain_sequences(state):
    """Paths back by doubling: map[t] first goes one step back from t, then two, four, ..."""
    case = state["case"]
    N, K, T = case["groups"], case["beams"], case["steps"]
    tokens = state["tokens"].view(T, N, K).long()
    parents = state["parents"].view(T, N, K).long()
    end, first = state["end_step"].long(), state["end_parent"].long()
    # beam of every hypothesis at every step before its end: known at t = end - 1, unknown (-1) earlier
    t = torch.arange(T, device="cuda")[:, None, None]
    beam = torch.where(t == end - 1, first, -1)
    hop = torch.cat([parents[1:], parents[:1]])  # leads from the beam at t + 1 to its parent at t
    reach = 1
    while reach < T:
        ahead = torch.cat([beam[reach:], torch.full_like(beam[:reach], -1)])
        beam = torch.where(beam >= 0, beam, torch.where(ahead >= 0, hop.gather(2, ahead.clamp(min=0)), -1))
        hop = hop.gather(2, torch.cat([hop[reach:], hop[:reach]]))  # leads from t + 2 * reach to t
        reach *= 2
    seq = torch.where(beam >= 0, tokens.gather(2, beam.clamp(min=0)), -1)
    seq = torch.where(t == end, state["end_token"].long(), seq)
    return {"tokens": seq.permute(1, 2, 0).int().contiguous(), "lens": (end + 1).int()}


def _activated(y, activation, scale):
    if activation == "relu":
        return torch.clamp(y, min=0)
    if activation == "sigmoid":
        return 1 / (1 + torch.exp(-y))
    if activation == "tanh":
        return scale * torch.tanh(y / scale)
    if activation == "gelu":
        return 0.5 * y * (1 + torch.erf(y / math.sqrt(2)))
    if activation == "silu":
        return y / (1 + torch.exp(-y))
    return y


def _plain_linear(state):
    case = state["case"]
    y = state["x"].float() @ state["weight"].float().t()
    if "bias" in state:
        y = y + state["bias"]
    y = _activated(y, case["activation"], case["scale"])
    if "residual" in state:
        y = y + state["residual"].float()
    return y.to(_DTYPES[case["out"]])


_PLAIN = {"step": _plain_step, "reorder": _plain_reorder, "sequences": _plain_sequences, "linear": _plain_linear}


# ---- the library's calls --------------------------------------------------------------------
_handles = []


def _sampler():
    from born_b200 import Sampler
    if not _handles:
        _handles.append(Sampler(device=0, max_batch=256, max_vocab=262144))
    return _handles[0]


def _call(state):
    """A decode loop runs over fixed buffers: the arguments of its calls are marshalled once."""
    from born_b200 import BeamConfig
    case, s = state["case"], _sampler()
    if case["op"] == "step":
        config = BeamConfig(temperature=case["temperature"], repetition_penalty=case["repetition"],
                            frequency_penalty=case["frequency"], presence_penalty=case["presence"],
                            stop_tokens=tuple(state["stops"]), keep_slots=case["keep_slots"])
        return s.prepare_beam_step(state["logits"], state["scores"], case["beams"], config=config,
                                   mask=state.get("mask"), history=state.get("history"))
    if case["op"] == "reorder":
        return s.prepare_beam_reorder(list(state["buffers"]), state["parents"], case["beams"], lens=state.get("lens"),
                                      position_dim=2)
    if case["op"] == "sequences":
        return s.prepare_beam_sequences(state["tokens"], state["parents"], state["end_step"], state["end_parent"],
                                        state["end_token"], case["beams"])
    return s.prepare_linear(state["x"], state["weight"], bias=state.get("bias"), residual=state.get("residual"),
                            activation=case["activation"], scale=case["scale"], out_dtype=_DTYPES[case["out"]])


def _own(state):
    if "call" not in state:
        state["call"] = _call(state)
    out = state["call"].run()
    if state["case"]["op"] == "reorder":
        return state["buffers"]
    if state["case"]["op"] == "step":
        names = ["parent", "token", "score"] + (["end_parent", "end_token", "end_score"] if state["stops"] else [])
        return {n: out[n] for n in names}
    return out


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------
def work(case):
    if case["op"] == "step":
        N, K, V = case["groups"], case["beams"], case["vocab"]
        rows = N if case["first"] else N * K  # a beam with a score of -inf has no candidates
        row = V * (4 if case["dtype"] == "f32" else 2) + 4 * case["history"] + (4 * ((V + 31) // 32) if case["mask"] else 0)
        return {"bytes": rows * row + N * K * (4 + 12 + (12 if case["stops"] else 0)), "flops": 4 * rows * V}
    if case["op"] == "reorder":
        N, K = case["groups"], case["beams"]
        row = case["buffers"] * case["planes"] * case["positions"] * case["width"] * (4 if case["dtype"] == "f32" else 2)
        dies = K * (1 - 1 / K) ** K  # rows taken over, of K parents drawn at random
        read = (K - dies) * (1 - (1 - 1 / K) ** dies)  # rows that they are read from
        return {"bytes": N * row * (dies + read) * (0.5 if case["ragged"] else 1.0) + 4 * N * K, "flops": 0}
    if case["op"] == "sequences":
        N, K, T = case["groups"], case["beams"], case["steps"]
        return {"bytes": N * K * (8 * T + 4 * T + 16), "flops": 0}
    M, H, V = case["rows"], case["hidden"], case["vocab"]
    out = 4 if case["out"] == "f32" else 2
    return {"bytes": 2 * M * H + 2 * V * H + M * V * out * (2 if case["residual"] else 1) + (4 * V if case["bias"] else 0),
            "flops": 2 * M * H * V}


# ---- the definitions in 64 bits -----------------------------------------------------------------
def _exact_step(case, state):
    N, K, V = case["groups"], case["beams"], case["vocab"]
    T = float(torch.tensor(case["temperature"], dtype=torch.float32))
    stops = set(state["stops"])
    parents, tokens, scores, ends = [], [], [], []
    for n in range(N):
        rows = slice(n * K, (n + 1) * K)
        part = {k: state[k][rows] for k in ("mask", "history") if k in state}
        z = _penalised(case, state["logits"][rows].float(), part).double() / T
        s = state["scores"][rows].double()
        flat = (s[:, None] + torch.log_softmax(z, dim=1)).reshape(-1)
        value, index = (v[:K * (len(stops) + 1)].tolist() for v in torch.sort(flat, descending=True, stable=True))
        ranked = [(v, i // V, i % V) for v, i in zip(value, index) if v > -math.inf]
        ended = [c for c in ranked[:K] if c[2] in stops]
        going = [c for c in ranked if c[2] not in stops][:K]
        rows_of = [None] * K
        if case["keep_slots"]:
            late = []
            for c in going:
                if rows_of[c[1]] is None:
                    rows_of[c[1]] = c
                else:
                    late.append(c)
            for r in range(K):
                if rows_of[r] is None and late:
                    rows_of[r] = late.pop(0)
        else:
            rows_of[:len(going)] = going
        rows_of = [c or (-math.inf, r, -1) for r, c in enumerate(rows_of)]
        ended += [(-math.inf, -1, -1)] * (K - len(ended))
        scores += [c[0] for c in rows_of]
        parents += [c[1] for c in rows_of]
        tokens += [c[2] for c in rows_of]
        ends.append(ended)
    out = {"parent": torch.tensor(parents, dtype=torch.int32), "token": torch.tensor(tokens, dtype=torch.int32),
           "score": torch.tensor(scores, dtype=torch.float64)}
    if stops:
        out["end_parent"] = torch.tensor([[c[1] for c in e] for e in ends], dtype=torch.int32)
        out["end_token"] = torch.tensor([[c[2] for c in e] for e in ends], dtype=torch.int32)
        out["end_score"] = torch.tensor([[c[0] for c in e] for e in ends], dtype=torch.float64)
    return out


def _exact_linear(case, state):
    if case["rows"] * case["hidden"] * case["vocab"] > 300_000_000_000:
        return None
    x, parts = state["x"].double(), []
    for at in range(0, case["vocab"], 16384):
        y = torch.matmul(x, state["weight"][at:at + 16384].double().T)
        if "bias" in state:
            y += state["bias"][at:at + 16384].double()
        a = case["activation"]
        if a == "relu":
            y = torch.where(y > 0, y, torch.zeros_like(y))
        elif a == "tanh":
            y = case["scale"] * (1 - 2 / (torch.exp(2 * y / case["scale"]) + 1))
        elif a in ("sigmoid", "silu"):
            y = (y if a == "silu" else 1.0) * torch.sigmoid(y)
        elif a == "gelu":
            y = 0.5 * y * torch.erfc(-y / 2 ** 0.5)
        if "residual" in state:
            y += state["residual"][:, at:at + 16384].double()
        parts.append(y)
    return torch.cat(parts, dim=1)


def exact(case, seed):
    """Definitions in 64 bits.  Reordered states and read-out sequences are moved, not computed."""
    if case["op"] == "step":
        return _exact_step(case, prepare(case, seed))
    if case["op"] == "linear":
        return _exact_linear(case, prepare(case, seed))
    return None
