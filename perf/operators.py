"""The quantised speaker registry's operators, as cases that can be timed and compared.

A registry holds one unit embedding per enrolled speaker in 8 or 4 bits a dimension. A
row x is stored as small integers w and one f32 scale 1 / |w|, so that it stands for the
unit vector w / |w|:

  8 bits   w = rint(127 x / max|x|)
  4 bits   per group g of 32 dimensions a 7-bit scale s_g = ceil(127 max_g|x| / max|x|)
           and codes c = rint(889 x / (max|x| s_g)) in -7 .. 7; w = c s_g

A slot that was never written, was cleared, or was given a row with an infinity or a NaN
is empty (its scale is NaN): it reads back as NaN, scores -inf and takes no part in a
posterior. Three operators work on it:

  enrol      rows are written to given slots (negative: skipped; the same slot twice: the
             last row stays) and read back as the unit vectors that the registry now holds
  score      cosines of a few queries with every row (a matrix-vector product with 8-bit or
             with grouped 4-bit weights)
  posterior  softmax(scale * cosine) over the enrolled rows: the log probability of each
             query's claimed speaker, the entropy, the log of the normaliser, and the k most
             probable speakers with their log probabilities (ranked by the cosine rounded
             to f32, equal ones by the lower slot)

`run` computes them from elementary torch operations, or, where `own` is true, calls
vd_b200.Registry.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parents[1] / "voice-detect.cpp_b200")
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one caller enrols while the service runs: a single embedding into a free slot
        {"name": "enrol_one", "op": "enrol", "bits": 8, "dim": 256, "rows": 1, "capacity": 1000,
         "type": "f32", "spread": True},
        # a bucket of clips embedded in one batch, padded rows skipped and a few speakers in it
        # twice; 192 dimensions as ECAPA gives, kept in f16 by the caller
        {"name": "enrol_bucket_f16", "op": "enrol", "bits": 8, "dim": 192, "rows": 4099,
         "capacity": 20000, "type": "f16", "spread": True},
        # a whole registry built at start-up, in order
        {"name": "enrol_registry_4bit", "op": "enrol", "bits": 4, "dim": 256, "rows": 100000,
         "capacity": 100000, "type": "f32", "spread": False},
        # one utterance against a team's small registry: latency alone
        {"name": "score_team", "op": "score", "bits": 8, "dim": 256, "rows": 777, "queries": 1,
         "type": "f32"},
        # a few test utterances against an impostor cohort, for score normalisation
        {"name": "score_cohort", "op": "score", "bits": 8, "dim": 512, "rows": 20011,
         "queries": 16, "type": "f32"},
        # one utterance against two million 4-bit rows: the registry's bytes are the cost
        {"name": "score_large_4bit", "op": "score", "bits": 4, "dim": 256, "rows": 2000003,
         "queries": 1, "type": "f32"},
        # open-set identification of one utterance in a small registry
        {"name": "posterior_team", "op": "posterior", "bits": 4, "dim": 192, "rows": 1000,
         "queries": 1, "k": 5, "scale": 30.0, "type": "f32"},
        # one utterance against a city-sized registry
        {"name": "posterior_one_4bit", "op": "posterior", "bits": 4, "dim": 256, "rows": 1000000,
         "queries": 1, "k": 5, "scale": 30.0, "type": "f32"},
        # the speakers of a meeting, one embedding each, against the benchmark's registry
        {"name": "posterior_meeting", "op": "posterior", "bits": 8, "dim": 256, "rows": 100000,
         "queries": 12, "k": 5, "scale": 30.0, "type": "bf16"},
        # an odd batch in between, with many alternatives
        {"name": "posterior_odd", "op": "posterior", "bits": 4, "dim": 300, "rows": 5003,
         "queries": 301, "k": 20, "scale": 20.0, "type": "f16"},
        # a batch job: the benchmark's 8192 embeddings against its 100,000 speakers, top 5
        {"name": "posterior_batch", "op": "posterior", "bits": 8, "dim": 256, "rows": 100000,
         "queries": 8192, "k": 5, "scale": 30.0, "type": "f32"},
        # the same batch against a 4-bit registry of CAM++'s 512 dimensions
        {"name": "posterior_batch_4bit", "op": "posterior", "bits": 4, "dim": 512, "rows": 50001,
         "queries": 4096, "k": 10, "scale": 30.0, "type": "f32"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["enrol", "score", "posterior", "posterior"])
    case = {"op": op, "bits": rng.choice([4, 8]), "dim": rng.choice([192, 256, 512, rng.randint(64, 512)]),
            "type": rng.choice(["f32", "f32", "f16", "bf16"])}
    if op == "enrol":
        case["rows"] = _log_int(rng, 1, 100000)
        case["capacity"] = case["rows"] + rng.randint(0, 20000)
        case["spread"] = rng.random() < 0.6
        return case
    if op == "score":
        case["queries"] = _log_int(rng, 1, 64)
        case["rows"] = _log_int(rng, 1, 2000000 // case["queries"])
        return case
    case["queries"] = _log_int(rng, 1, 8192)
    case["rows"] = _log_int(rng, 1, min(1000000, 819200000 // case["queries"] * 256 // case["dim"]))
    case["k"] = rng.choice([0, 1, 5, 5, 8, 10, rng.randint(1, 64)])
    case["scale"] = round(rng.uniform(8.0, 40.0), 2)
    return case


# --------------------------------------------------------------------------- the inputs
def _embeddings(n, dim, gen):
    """n embeddings as an encoder leaves them: a common offset, a speaker's own direction,
    and a length of its own; about one row in five hundred repeats another."""
    centre = torch.randn(dim, generator=gen, device="cuda")
    x = torch.randn(n, dim, generator=gen, device="cuda") + 0.3 * centre
    x *= torch.rand(n, 1, generator=gen, device="cuda") * 2 + 0.2
    twice = torch.rand(n, generator=gen, device="cuda") < 0.002
    other = torch.randint(0, n, (n,), generator=gen, device="cuda")
    return torch.where(twice[:, None], x[other], x)


def _inputs(case, seed):
    """The case's embeddings, slots, queries and labels, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    n, dim = case["rows"], case["dim"]
    x = _embeddings(n, dim, gen)
    if case["op"] == "enrol":
        got = {"x": x.to(_TYPES[case["type"]]), "slots": None}
        if case["spread"]:
            slots = torch.randperm(case["capacity"], generator=gen, device="cuda")[:n]
            if n > 1:
                again = torch.rand(n, generator=gen, device="cuda") < 0.01
                slots = torch.where(again, slots.roll(n // 2), slots)
                slots[torch.rand(n, generator=gen, device="cuda") < 0.01] = -1
            got["slots"] = slots.to(torch.int32)
        return got
    m = case["queries"]
    empty = torch.rand(n, generator=gen, device="cuda") < 0.01
    who = torch.randint(0, n, (m,), generator=gen, device="cuda")
    noise = torch.randn(m, dim, generator=gen, device="cuda") * x.std()
    known = torch.rand(m, 1, generator=gen, device="cuda") < 0.75
    q = torch.where(known, x[who] + noise, noise)
    got = {"x": x, "empty": torch.nonzero(empty).flatten().to(torch.int32),
           "q": q.to(_TYPES[case["type"]])}
    if case["op"] == "posterior":
        claim = torch.rand(m, generator=gen, device="cuda")
        label = torch.where(claim < 0.8, who, torch.randint(0, n, (m,), generator=gen, device="cuda"))
        got["labels"] = torch.where(claim > 0.97, torch.full_like(label, -1), label).to(torch.int32)
    return got


# ----------------------------------------------------------------------- the plain form
def _quantise(x, bits):
    """(codes int8 [n][dim], group scales uint8 [n][groups] or None, scale f32 [n]). The
    quotients are taken in 64 bits: one next to a half has to round the right way."""
    bad = ~torch.isfinite(x).all(1)
    v = torch.where(bad[:, None], torch.zeros_like(x), x).double()
    n, dim = v.shape
    top = v.abs().amax(1, keepdim=True)
    safe = torch.where(top > 0, top, torch.ones_like(top))
    if bits == 8:
        w = torch.round(v * 127 / safe)
        codes, group = w.to(torch.int8), None
    else:
        pad = torch.nn.functional.pad(v, (0, -dim % 32)).reshape(n, -1, 32)
        s = torch.ceil(pad.abs().amax(2) * 127 / safe)
        c = torch.round(pad * 889 / (safe * s.clamp_min(1))[:, :, None])
        codes = c.reshape(n, -1)[:, :dim].to(torch.int8)
        group = s.to(torch.uint8)
        w = (c * s[:, :, None]).reshape(n, -1)
    square = (w * w).sum(1)
    scale = torch.where(square > 0, square.rsqrt(), torch.zeros_like(square)).float()
    return codes, group, torch.where(bad, torch.full_like(scale, math.nan), scale)


def _whole(codes, group):
    """The integers w, as f32 (exact)."""
    w = codes.float()
    if group is not None:
        w = w * group.float().repeat_interleave(32, 1)[:, :w.shape[1]]
    return w


def _enrol(state):
    x, slots = state["x"], state["slots"]
    n, capacity = len(x), state["capacity"]
    if slots is None:
        slots = torch.arange(n, device=x.device)
    slots = slots.long()
    order = torch.arange(n, device=x.device)
    keep = slots >= 0
    # the last row of each slot (row `capacity` takes what is skipped)
    place = torch.where(keep, slots, torch.full_like(slots, capacity))
    last = torch.full((capacity + 1,), -1, device=x.device).scatter_reduce(0, place, order, "amax")
    stays = keep & (last[place] == order)
    codes, group, scale = _quantise(x.float(), state["bits"])
    state["codes"][place[stays]] = codes[stays]
    state["scale"][place[stays]] = scale[stays]
    if group is not None:
        state["group"][place[stays]] = group[stays]
    # read back what these slots now hold
    at = place.clamp_max(capacity - 1)
    value = _whole(state["codes"][at], group if group is None else state["group"][at])
    value = value * state["scale"][at][:, None]
    return torch.where(keep[:, None], value, torch.full_like(value, math.nan))


def _score(state):
    q = state["q"].float()
    length = q.norm(dim=1, keepdim=True)
    unit = torch.where(length > 0, q / length, torch.zeros_like(q))
    scale = state["scale"]
    empty = torch.isnan(scale)
    rows = _whole(state["codes"], state["group"]) * torch.where(empty, torch.zeros_like(scale), scale)[:, None]
    return (unit @ rows.T).masked_fill(empty, -math.inf)


def _posterior(state):
    # in 64 bits throughout: near cosines have to be told apart, the sums run over a whole
    # registry, and a confident posterior's log probability and entropy are next to 0
    q = state["q"].double()
    w = _whole(state["codes"], state["group"]).double()
    length = q.norm(dim=1)[:, None] * w.norm(dim=1)
    cos = q @ w.T / torch.where(length > 0, length, torch.ones_like(length))
    empty = torch.isnan(state["scale"])
    z = (cos * state["temperature"]).masked_fill(empty, -math.inf)
    top = z.amax(1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    e = torch.exp(z - top)
    total = e.sum(1)
    lse = torch.log(total) + top[:, 0]
    entropy = torch.log(total) - (e * torch.where(empty, torch.zeros_like(z), z - top)).sum(1) / total
    entropy = torch.where(total > 0, entropy, torch.zeros_like(entropy))
    label = state["labels"].long()
    none = (label < 0) | (label >= z.shape[1])
    claimed = z.gather(1, label.clamp(0, z.shape[1] - 1)[:, None])[:, 0]
    log_prob = torch.where(none | torch.isinf(claimed), torch.full_like(lse, -math.inf), claimed - lse)
    # one whole-number key a score: the f32 cosine's order above, the lower slot below
    bits = (cos.float() + 0.0).view(torch.int32).long()
    key = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).masked_fill(empty, -2 ** 31)
    slot = torch.arange(z.shape[1], device=z.device)
    k = min(state["k"], z.shape[1])
    best = (key * 2 ** 32 + (2 ** 32 - 1 - slot)).topk(k, dim=1).values
    index = 2 ** 32 - 1 - (best & (2 ** 32 - 1))
    found = (best >> 32) > -2 ** 31
    alt = torch.where(found, z.gather(1, index) - lse[:, None], torch.full_like(lse, -math.inf)[:, None])
    index = torch.where(found, index, torch.full_like(index, -1))
    more = state["k"] - k
    return {"log_prob": log_prob.float(), "entropy": entropy.float(), "lse": lse.float(),
            "index": torch.nn.functional.pad(index, (0, more), value=-1).to(torch.int32),
            "alt_log_prob": torch.nn.functional.pad(alt.float(), (0, more), value=-math.inf)}


# ------------------------------------------------------------------------------ the calls
def prepare(case, seed):
    got = _inputs(case, seed)
    if case["op"] == "enrol":
        state = {"op": "enrol", "x": got["x"], "slots": got["slots"], "bits": case["bits"],
                 "capacity": case["capacity"]}
        rows = case["capacity"]
    else:
        state = {"op": case["op"], "q": got["q"]}
        rows = case["rows"]
        if case["op"] == "posterior":
            state |= {"labels": got["labels"], "k": case["k"], "temperature": case["scale"]}
    if own:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        import vd_b200
        registry = vd_b200.Registry(rows, case["dim"], bits=case["bits"])
        if case["op"] != "enrol":
            registry.write(got["x"])
            registry.clear(got["empty"])
        return state | {"registry": registry}
    if case["op"] == "enrol":
        state["codes"] = torch.zeros(rows, case["dim"], dtype=torch.int8, device="cuda")
        state["group"] = torch.zeros(rows, (case["dim"] + 31) // 32, dtype=torch.uint8, device="cuda")
        state["scale"] = torch.full((rows,), math.nan, device="cuda")
    else:
        state["codes"], state["group"], state["scale"] = _quantise(got["x"], case["bits"])
        state["scale"][got["empty"].long()] = math.nan
    return state


def run(state):
    if not own:
        return {"enrol": _enrol, "score": _score, "posterior": _posterior}[state["op"]](state)
    registry = state["registry"]
    if state["op"] == "enrol":
        registry.write(state["x"], state["slots"])
        return registry.read(state["slots"], n=len(state["x"]))
    if state["op"] == "score":
        return registry.score(state["q"])
    p = registry.posterior(state["q"], state["labels"], k=state["k"], scale=state["temperature"])
    return {"log_prob": p.log_prob, "entropy": p.entropy, "lse": p.lse, "index": p.index,
            "alt_log_prob": p.alt_log_prob}


def work(case):
    n, dim = case["rows"], case["dim"]
    width = 4 if case["type"] == "f32" else 2
    row = dim + 4 if case["bits"] == 8 else (dim + 1) // 2 + (dim + 31) // 32 + 4
    if case["op"] == "enrol":
        slots = 4 * n if case["spread"] else 0
        # the embeddings in, the rows written, the unit vectors out
        return {"bytes": n * dim * width + n * row + n * dim * 4 + slots, "flops": 8 * n * dim}
    m = case["queries"]
    if case["op"] == "score":
        return {"bytes": n * row + m * dim * width + 4 * m * n, "flops": 2 * m * n * dim}
    return {"bytes": n * row + m * (dim * width + 4) + m * (12 + 8 * case["k"]),
            "flops": 2 * m * n * dim + 6 * m * n}


# --------------------------------------------------------------- the definition in 64 bits
def _unit_rows(x, bits):
    """What the registry holds of the rows of x, as unit vectors in 64 bits, and which rows
    it holds at all."""
    x = x.to(torch.float64)
    held = torch.isfinite(x).all(dim=-1)
    x = torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0)
    peak = torch.linalg.vector_norm(x, ord=math.inf, dim=-1)
    peak[peak == 0] = 1.0
    w = torch.empty_like(x)
    if bits == 8:
        torch.round(127.0 * x / peak[:, None], out=w)
    else:
        for lo in range(0, x.shape[1], 32):
            part = x[:, lo:lo + 32]
            s = torch.ceil(127.0 * torch.linalg.vector_norm(part, ord=math.inf, dim=-1) / peak)
            step = torch.where(s > 0, peak * s, torch.ones_like(s))
            w[:, lo:lo + 32] = torch.round(889.0 * part / step[:, None]) * s[:, None]
    size = torch.linalg.vector_norm(w, dim=-1)
    size[size == 0] = 1.0
    return w / size[:, None], held


def exact(case, seed):
    got = _inputs(case, seed)
    unit, held = _unit_rows(got["x"], case["bits"])
    if case["op"] == "enrol":
        unit[~held] = math.nan
        if got["slots"] is None:
            return unit
        slots = got["slots"].tolist()
        last = {s: i for i, s in enumerate(slots)}
        out = unit[torch.tensor([last[s] for s in slots], device=unit.device)]
        out[got["slots"] < 0] = math.nan
        return out
    held[got["empty"].long()] = False
    q = got["q"].to(torch.float64)
    size = torch.linalg.vector_norm(q, dim=-1, keepdim=True)
    q = q / torch.where(size == 0, torch.ones_like(size), size)
    if case["op"] == "score":
        out = q @ unit.mT
        out[:, ~held] = -math.inf
        return out
    slots = torch.nonzero(held).flatten()
    unit = unit[slots]
    parts = []
    for lo in range(0, len(q), 1024):
        cos = q[lo:lo + 1024] @ unit.mT
        logits = case["scale"] * cos
        lse = torch.logsumexp(logits, dim=-1)
        log_p = logits - lse[:, None]
        entropy = -(log_p.exp() * log_p).sum(dim=-1)
        label = got["labels"][lo:lo + 1024].long()
        known = (label >= 0) & held[label.clamp_min(0)]
        at = torch.searchsorted(slots, label).clamp_max(max(0, len(slots) - 1))
        claim = torch.full_like(lse, -math.inf)
        claim[known] = log_p[known, at[known]]
        k = min(case["k"], len(slots))
        order = torch.sort(cos.float(), dim=-1, descending=True, stable=True).indices[:, :k]
        index = torch.full((len(cos), case["k"]), -1, dtype=torch.int32, device=cos.device)
        alt = torch.full((len(cos), case["k"]), -math.inf, dtype=torch.float64, device=cos.device)
        index[:, :k] = slots[order].to(torch.int32)
        alt[:, :k] = log_p.gather(1, order)
        parts.append((claim, entropy, lse, index, alt))
    names = ("log_prob", "entropy", "lse", "index", "alt_log_prob")
    return {name: torch.cat([p[i] for p in parts]) for i, name in enumerate(names)}
