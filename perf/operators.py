"""The paged cache's operators on their real range, through the package's public entry points.

A case is a dict of plain values; lengths follow from the case alone (``batch`` seeds them), tensors
from the seed. Kinds of call (``op``):

- ``attend``: ``paged_attention``, rows of new tokens against the pages that hold their sequences'
  keys, from single decoded tokens to chunks of a long prompt.
- ``append``: ``paged_append``, the new tokens' q and k rotated and their k and v written into pages.
- ``rotary``: ``rotary``, rotary positions of either layout on part of the head or all of it; with
  ``train`` the gradient too.
- ``pages``: ``copy_pages``, pages copied within a cache of several layers (forked sequences that
  need a last page of their own, a pool compacted into its low pages).

Head geometries are those of the package's other measured cases (32:8 and 16:8 heads of 128, 8:2 of
256, 12:12 of 64).
"""

from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def listed() -> list[dict]:
    gqa128 = {"hq": 32, "hkv": 8, "d": 128}
    gqa256 = {"hq": 8, "hkv": 2, "d": 256}
    return [
        # a quiet server: four users, one token each, short histories; latency counts
        {"name": "decode_small", "op": "attend", **gqa128, "page": 16, "steps": 4, "chunks": 0, "new_lo": 1,
         "new_hi": 1, "lo": 100, "hi": 600, "window": -1, "causal": True, "batch": 1},
        # a busy server's decoding step: 64 users at ordinary to long histories
        {"name": "decode_batch", "op": "attend", **gqa128, "page": 64, "steps": 64, "chunks": 0, "new_lo": 1,
         "new_hi": 1, "lo": 512, "hi": 8192, "window": -1, "causal": True, "batch": 2},
        # few users with very long documents, heads of 256 as in the hybrid encoder's attention layer
        {"name": "decode_long", "op": "attend", **gqa256, "page": 128, "steps": 3, "chunks": 0, "new_lo": 1,
         "new_hi": 1, "lo": 60000, "hi": 131072, "window": -1, "causal": True, "batch": 3},
        # a chunk of a long prompt against what is cached of it: the largest attention call
        {"name": "chunk_long", "op": "attend", **gqa128, "page": 64, "steps": 0, "chunks": 1, "new_lo": 2048,
         "new_hi": 2048, "lo": 16384, "hi": 16384, "window": -1, "causal": True, "batch": 4},
        # one step of a server that mixes decoding users with two prompts' ragged chunks, windowed layers
        {"name": "mixed_window", "op": "attend", "hq": 12, "hkv": 12, "d": 64, "page": 16, "steps": 30, "chunks": 2,
         "new_lo": 200, "new_hi": 777, "lo": 800, "hi": 6000, "window": 1023, "causal": True, "batch": 5},
        # a decoding step's new tokens: rotated and written, one row per user
        {"name": "append_step", "op": "append", **gqa128, "page": 16, "steps": 128, "chunks": 0, "new_lo": 1,
         "new_hi": 1, "lo": 64, "hi": 4096, "rot": 128, "interleaved": False, "theta": 500000.0, "scale": 1.0,
         "batch": 6},
        # prompts entering the cache, a quarter of each head rotated in pairs
        {"name": "append_prompts", "op": "append", **gqa256, "page": 64, "steps": 0, "chunks": 5, "new_lo": 2500,
         "new_hi": 8000, "lo": 8000, "hi": 20000, "rot": 64, "interleaved": True, "theta": 10000000.0,
         "scale": 1.0, "batch": 7},
        # a decoding step's rows far into a long context, the amplitude scaled as long contexts have it
        {"name": "rotary_step", "op": "rotary", "tokens": 64, "heads": 40, "d": 128, "rot": 128, "interleaved": False,
         "type": "bfloat16", "span": 131072, "theta": 500000.0, "scale": 1.1386, "train": False},
        # training on long documents: rotation and its gradient
        {"name": "rotary_train", "op": "rotary", "tokens": 16384, "heads": 32, "d": 128, "rot": 128,
         "interleaved": False, "type": "bfloat16", "span": 8192, "theta": 160000.0, "scale": 1.0, "train": True},
        # a ragged packed batch in 32 bits, part of the head in pairs, positions up to a million
        {"name": "rotary_partial", "op": "rotary", "tokens": 30011, "heads": 8, "d": 256, "rot": 64,
         "interleaved": True, "type": "float32", "span": 1000000, "theta": 10000000.0, "scale": 1.0, "train": False},
        # eight sequences forked inside a page: each gets a copy of the shared last page in every layer
        {"name": "fork_step", "op": "pages", "layers": 22, "pool": 256, "page": 16, "hkv": 8, "d": 128, "pairs": 8,
         "batch": 8},
        # a pool compacted: scattered pages move into the freed low ones, in every layer
        {"name": "compact_pool", "op": "pages", "layers": 12, "pool": 1024, "page": 32, "hkv": 8, "d": 128,
         "pairs": 400, "batch": 9},
    ]


def _log(rng, lo: float, hi: float) -> int:
    return max(int(lo), min(int(hi), round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    """One more case of the listed ones' ranges (sizes over their logarithm)."""
    batch = rng.randrange(1 << 30)
    hq, hkv, d = rng.choice(((32, 8, 128), (16, 8, 128), (16, 16, 128), (8, 2, 256), (12, 12, 64), (20, 4, 64)))
    heads = {"hq": hq, "hkv": hkv, "d": d, "page": rng.choice((16, 32, 48, 64, 128, 256)), "batch": batch}
    window = rng.choice((-1, -1, -1, _log(rng, 64, 4096)))
    kind = rng.randrange(8)
    if kind in (0, 1):  # decoding steps, one token each, or a few drafted ones to check
        top = _log(rng, 1000, 16384)
        return {"op": "attend", **heads, "steps": _log(rng, 1, 64), "chunks": rng.choice((0, 0, 3)), "new_lo": 2,
                "new_hi": 9, "lo": rng.randint(1, 600), "hi": top, "window": window, "causal": True}
    if kind == 2:  # long documents
        return {"op": "attend", **heads, "steps": rng.randint(1, 3), "chunks": 0, "new_lo": 1, "new_hi": 1,
                "lo": 20000, "hi": _log(rng, 30000, 100000), "window": window, "causal": True}
    if kind == 3:  # chunks of prompts beside decoding users
        new = _log(rng, 16, 1024)
        return {"op": "attend", **heads, "steps": rng.choice((0, rng.randint(1, 24))), "chunks": rng.randint(1, 3),
                "new_lo": max(1, new // 3), "new_hi": new, "lo": new, "hi": new + _log(rng, 16, 6000),
                "window": window, "causal": rng.random() < 0.8}
    inner = {"rot": rng.choice((d, d // 2, d // 4, 16)), "interleaved": rng.random() < 0.5,
             "theta": rng.choice((10000.0, 160000.0, 500000.0, 10000000.0)), "scale": rng.choice((1.0, 1.0, 1.2079))}
    if kind == 4:  # new tokens into pages
        new = _log(rng, 1, 4000)
        return {"op": "append", **heads, **inner, "steps": _log(rng, 1, 128), "chunks": rng.randint(0, 4),
                "new_lo": max(1, new // 4), "new_hi": new, "lo": new, "hi": new + _log(rng, 16, 8000)}
    if kind in (5, 6):  # rotary positions, forward or trained
        return {"op": "rotary", "tokens": _log(rng, 1, 16000), "heads": rng.choice((1, 5, 8, 12, 32)), "d": d, **inner,
                "type": rng.choice(("bfloat16", "bfloat16", "float16", "float32")), "span": _log(rng, 512, 1000000),
                "train": rng.random() < 0.5}
    pool = _log(rng, 16, 700)
    return {"op": "pages", "layers": rng.randint(1, 22), "pool": pool, "page": rng.choice((16, 32, 48)),
            "hkv": rng.choice((2, 8, 12)), "d": rng.choice((64, 128)), "pairs": rng.randint(1, pool // 2), "batch": batch}


# ----------------------------------------------------------------------------- sizes


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(new tokens, keys with them) of each sequence: the decoding ones, then the chunks."""
    rng = random.Random(case["batch"])
    new, keys = [], []
    for i in range(case["steps"] + case["chunks"]):
        n = 1 if i < case["steps"] else rng.randint(case["new_lo"], case["new_hi"])
        new.append(n)
        keys.append(max(n, rng.randint(case["lo"], case["hi"])))
    return new, keys


def _pairs(case: dict) -> tuple[list[int], list[int]]:
    """Pages copied and where to: distinct pages, no target among the sources."""
    order = list(range(case["pool"]))
    random.Random(case["batch"]).shuffle(order)
    n = case["pairs"]
    return order[:n], order[n:2 * n]


def _reach(n: int, keys: int, window: int, causal: bool) -> int:
    """(row, key) pairs that `n` new rows at the end of `keys` keys attend to."""
    total = 0
    for r in range(n):
        at = keys - n + r
        total += (at + 1 if causal else keys) - (max(0, at - window) if window >= 0 else 0)
    return total


def work(case: dict) -> dict:
    if case["op"] == "rotary":
        size = 4 if case["type"] == "float32" else 2
        passes = 2 if case["train"] else 1
        n = case["tokens"] * case["heads"]
        return {"bytes": passes * (2 * n * case["d"] * size + 8 * case["tokens"]), "flops": passes * 3 * n * case["rot"]}
    if case["op"] == "pages":
        page = case["page"] * case["hkv"] * case["d"] * 2
        return {"bytes": 2 * 2 * case["layers"] * case["pairs"] * page, "flops": 0}
    new, keys = _lengths(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "append":
        return {"bytes": 2 * sum(new) * (hq + 2 * hkv) * d * 2, "flops": 3 * sum(new) * (hq + hkv) * case["rot"]}
    # keys that some row of the sequence reaches are read once, q read and the output written once
    first = [max(0, k - n - case["window"]) if case["window"] >= 0 else 0 for n, k in zip(new, keys)]
    read = sum(k - f for k, f in zip(keys, first))
    return {"bytes": 2 * read * hkv * d * 2 + 2 * sum(new) * hq * d * 2,
            "flops": 4 * d * hq * sum(_reach(n, k, case["window"], case["causal"]) for n, k in zip(new, keys))}


# ----------------------------------------------------------------------------- inputs


def _randn(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _bounds(lengths: list[int]) -> torch.Tensor:
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _inverse_frequencies(rot: int, theta: float) -> torch.Tensor:
    return (theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().cuda()


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "rotary":
        n, dtype = case["tokens"], TYPES[case["type"]]
        # rows of a projection, as a layer hands them on, and a packed batch's positions
        state["x"] = _randn(gen, n, case["heads"], case["d"], dtype=dtype).requires_grad_(case["train"])
        state["grad"] = _randn(gen, n, case["heads"], case["d"], dtype=dtype) if case["train"] else None
        state["positions"] = torch.randint(0, case["span"], (n,), generator=gen, device="cuda")
        state["inv_freq"] = _inverse_frequencies(case["rot"], case["theta"])
        return state
    if case["op"] == "pages":
        shape = (case["layers"], case["pool"], case["page"], case["hkv"], case["d"])
        state["k"], state["v"] = _randn(gen, *shape), _randn(gen, *shape)
        state["src"], state["dst"] = _pairs(case)
        return state
    new, keys = _lengths(case)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    # a pool that has served for a while: every sequence's pages lie scattered over it
    used = [(k + page - 1) // page for k in keys]
    pool = sum(used) + 8
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(keys), max(used)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    state.update(new=new, keys=keys, max_new=max(new), max_keys=max(keys), table=table.cuda(), cu=_bounds(new),
                 lens=torch.tensor(keys, dtype=torch.int32, device="cuda"),
                 k_pages=_randn(gen, pool, page, hkv, d), v_pages=_randn(gen, pool, page, hkv, d))
    state["q"] = _randn(gen, sum(new), hq, d)
    if case["op"] == "append":  # k and v as views of one projection, as a layer has them
        rows = _randn(gen, sum(new), 2 * hkv, d)
        state["k"], state["v"] = rows[:, :hkv], rows[:, hkv:]
        state["inv_freq"] = _inverse_frequencies(case["rot"], case["theta"])
    return state


# ----------------------------------------------------------------------------- one pass


def run(state: dict):
    return (_own if own else _plain)[state["case"]["op"]](state, state["case"])


def _own_attend(s, case):
    import packed_encoders_amd as pe

    return pe.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["lens"], s["max_new"],
                              max_seqlen_k=s["max_keys"], window=(case["window"], -1), causal=case["causal"])


def _own_append(s, case):
    import packed_encoders_amd as pe

    q = pe.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["lens"], q=s["q"],
                        inv_freq=s["inv_freq"], interleaved=case["interleaved"], rope_scale=case["scale"])
    return q, s["k_pages"], s["v_pages"]


def _own_rotary(s, case):
    import packed_encoders_amd as pe

    y = pe.rotary(s["x"], s["positions"], s["inv_freq"], interleaved=case["interleaved"], scale=case["scale"])
    if not case["train"]:
        return y
    return y.detach(), torch.autograd.grad(y, s["x"], s["grad"])[0]


def _own_pages(s, case):
    import packed_encoders_amd as pe

    pe.copy_pages((s["k"], s["v"]), s["src"], s["dst"])
    return s["k"], s["v"]


_own = {"attend": _own_attend, "append": _own_append, "rotary": _own_rotary, "pages": _own_pages}


def _gather(pages, table, i: int, keys: int, page: int):
    """A sequence's rows of a cache, in order: [keys, heads, d]."""
    used = (keys + page - 1) // page
    return pages.index_select(0, table[i, :used].long()).flatten(0, 1)[:keys]


def _plain_attend(s, case):
    hq, hkv, d, page, window = case["hq"], case["hkv"], case["d"], case["page"], case["window"]
    out = torch.empty_like(s["q"])
    first = 0
    for i, (n, keys) in enumerate(zip(s["new"], s["keys"])):
        k = _gather(s["k_pages"], s["table"], i, keys, page).float().permute(1, 2, 0).contiguous()  # [hkv, d, keys]
        v = _gather(s["v_pages"], s["table"], i, keys, page).float().transpose(0, 1).contiguous()  # [hkv, keys, d]
        for r0 in range(0, n, 512):  # some rows at a time: the scores are in memory
            m = min(512, n - r0)
            q = s["q"][first + r0:first + r0 + m].float().view(m, hkv, hq // hkv, d).permute(1, 2, 0, 3)
            scores = torch.matmul(q.reshape(hkv, -1, d), k).view(hkv, hq // hkv, m, keys) * d ** -0.5
            at = torch.arange(keys - n + r0, keys - n + r0 + m, device="cuda")[:, None]
            key = torch.arange(keys, device="cuda")[None, :]
            allowed = torch.ones(m, keys, dtype=torch.bool, device="cuda")
            if case["causal"]:
                allowed = allowed & (key <= at)
            if window >= 0:
                allowed = allowed & (at - key <= window)
            scores = scores.masked_fill(~allowed, -math.inf)
            p = torch.exp(scores - scores.amax(-1, keepdim=True))
            o = torch.matmul(p.view(hkv, -1, keys), v).view(hkv, hq // hkv, m, d) / p.sum(-1, keepdim=True)
            out[first + r0:first + r0 + m] = o.permute(2, 0, 1, 3).reshape(m, hq, d).to(out.dtype)
        first += n
    return out


def _turn(x, positions, inv_freq, interleaved: bool, scale: float, sign: float = 1.0):
    """Rotated rows in 32 bits of x [tokens, heads, d]; angles in 64 (positions reach far)."""
    angle = positions.double()[:, None] * inv_freq.double()[None, :]
    cos, sin = (angle.cos() * scale).float()[:, None], (angle.sin() * (sign * scale)).float()[:, None]
    xf, half = x.float(), inv_freq.numel()
    out = xf.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    out[..., a] = xf[..., a] * cos - xf[..., b] * sin
    out[..., b] = xf[..., b] * cos + xf[..., a] * sin
    return out


def _plain_append(s, case):
    at = torch.cat([torch.arange(k - n, k, device="cuda") for n, k in zip(s["new"], s["keys"])])
    seq = torch.cat([torch.full((n,), i, device="cuda") for i, n in enumerate(s["new"])])
    page, slot = s["table"][seq, at // case["page"]].long(), at % case["page"]
    turn = (at, s["inv_freq"], case["interleaved"], case["scale"])
    q, k = _turn(s["q"], *turn).to(s["q"].dtype), _turn(s["k"], *turn).to(s["k"].dtype)
    s["k_pages"][page, slot] = k
    s["v_pages"][page, slot] = s["v"]
    return q, s["k_pages"], s["v_pages"]


def _plain_rotary(s, case):
    x = s["x"].detach()
    turn = (s["positions"], s["inv_freq"], case["interleaved"], case["scale"])
    y = _turn(x, *turn).to(x.dtype)
    if not case["train"]:
        return y
    return y, _turn_back(s["grad"], *turn).to(x.dtype)


def _turn_back(g, positions, inv_freq, interleaved: bool, scale: float):
    """The gradient of ``_turn``: the rotation by the opposite angle."""
    return _turn(g, positions, inv_freq, interleaved, scale, -1.0)


def _plain_pages(s, case):
    src, dst = torch.tensor(s["src"], device="cuda"), torch.tensor(s["dst"], device="cuda")
    for pages in (s["k"], s["v"]):
        pages[:, dst] = pages[:, src]
    return s["k"], s["v"]


_plain = {"attend": _plain_attend, "append": _plain_append, "rotary": _plain_rotary, "pages": _plain_pages}


# ----------------------------------------------------------------------------- the definition in 64 bits


def _exact_rotation(x, positions, inv_freq, interleaved: bool, scale: float, back: bool = False):
    """Each pair (a, b) as the complex number a + ib, times scale * exp(i angle)."""
    r = inv_freq.numel()
    angle = positions.double().view(-1, 1, 1) * inv_freq.double()
    factor = torch.polar(torch.full_like(angle, float(scale)), -angle if back else angle)
    xd = x.double()
    if interleaved:
        pairs = xd[..., :2 * r].unflatten(-1, (r, 2))
        z = torch.complex(pairs[..., 0], pairs[..., 1]) * factor
        turned = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(xd[..., :r], xd[..., r:2 * r]) * factor
        turned = torch.cat((z.real, z.imag), -1)
    return torch.cat((turned, xd[..., 2 * r:]), -1)


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "pages":
        return None  # nothing is computed
    if case["op"] == "rotary":
        turn = (s["positions"], s["inv_freq"], case["interleaved"], case["scale"])
        y = _exact_rotation(s["x"].detach(), *turn)
        return (y, _exact_rotation(s["grad"], *turn, back=True)) if case["train"] else y
    if case["op"] == "append":
        k_pages, v_pages, q_rows, first = s["k_pages"].double(), s["v_pages"].double(), [], 0
        for i, (n, keys) in enumerate(zip(s["new"], s["keys"])):
            at = torch.arange(keys - n, keys, device="cuda")
            turn = (at, s["inv_freq"], case["interleaved"], case["scale"])
            place = s["table"][i].long()[at // case["page"]] * case["page"] + at % case["page"]
            q_rows.append(_exact_rotation(s["q"][first:first + n], *turn))
            k_pages.flatten(0, 1)[place] = _exact_rotation(s["k"][first:first + n], *turn)
            v_pages.flatten(0, 1)[place] = s["v"][first:first + n].double()
            first += n
        return torch.cat(q_rows), k_pages, v_pages
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group, page, first = case["hq"] // case["hkv"], case["page"], 0
    for i, (n, keys) in enumerate(zip(s["new"], s["keys"])):
        place = (s["table"][i].long()[:, None] * page + torch.arange(page, device="cuda")).flatten()[:keys]
        far = (torch.arange(n, device="cuda") + keys - n)[:, None] - torch.arange(keys, device="cuda")[None, :]
        hidden = (far < 0) if case["causal"] else torch.zeros_like(far, dtype=torch.bool)
        if case["window"] >= 0:
            hidden = hidden | (far > case["window"])
        for h in range(case["hkv"]):
            k = s["k_pages"][:, :, h].flatten(0, 1)[place].double()
            v = s["v_pages"][:, :, h].flatten(0, 1)[place].double()
            for g in range(h * group, (h + 1) * group):
                scores = s["q"][first:first + n, g].double() @ k.t().contiguous() / math.sqrt(case["d"])
                weights = torch.softmax(scores.masked_fill_(hidden, -math.inf), -1)
                out[first:first + n, g] = weights @ v
        first += n
    return out
