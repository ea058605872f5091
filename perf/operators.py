"""Operators of serving and training next to the sliding-window attention, as cases to measure.

Four operators: rotary positions with several axes (forward and backward), the append of new
tokens' keys and values to a paged cache, the attention of one new token over that cache, and the
eviction of the cache's least attended entries.  ``run`` computes them in elementary torch
operations, or with ``own`` through the framework's entry points.
"""
import importlib
import math

import torch

own = False

PKG = "flashattention-gpt-oss-finetuning_b200"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _pkg(name):
    return importlib.import_module(f"{PKG}.{name}")


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------

def listed():
    return [
        # a fine-tuning step's rotation of q and k, and of their gradients, at the GPT-OSS layer
        dict(name="rotary-train-layer", op="rotary", dtype="bf16", batch=4, hq=64, hkv=8, length=4096, dim=64,
             axes=1, rot=64, interleaved=False, train=True, first=0),
        # the same with time, height and width axes: ragged length, large heads
        dict(name="rotary-train-3axis", op="rotary", dtype="f16", batch=8, hq=32, hkv=4, length=3000, dim=128,
             axes=3, rot=128, interleaved=False, train=True, first=0),
        # a short image prompt far into a conversation, neighbouring pairs, part of the head rotated
        dict(name="rotary-prompt-far", op="rotary", dtype="bf16", batch=1, hq=64, hkv=8, length=257, dim=64,
             axes=3, rot=48, interleaved=True, train=False, first=120000),
        # one decoding step of a batch: rotate q and k, write k and v to their pages
        dict(name="append-step", op="append", dtype="bf16", batch=64, hq=64, hkv=8, dim=64, page=64, new_min=1,
             new_max=1, old_min=100, old_max=4096, axes=1, track=False),
        # prompts of different lengths, packed, written behind a shared start
        dict(name="append-prompts", op="append", dtype="f16", batch=8, hq=32, hkv=4, dim=128, page=32, new_min=501,
             new_max=3000, old_min=0, old_max=64, axes=3, track=True),
        # the sliding-window layer of one conversation: the smallest call there is
        dict(name="decode-one-window", op="decode", dtype="bf16", batch=1, hq=64, hkv=8, dim=64, page=64, len_min=4096,
             len_max=4096, window=128, sinks=4, logits=True, weigh=False),
        # the same layer for a full serving batch
        dict(name="decode-batch-window", op="decode", dtype="bf16", batch=256, hq=64, hkv=8, dim=64, page=64, len_min=1,
             len_max=4096, window=128, sinks=4, logits=True, weigh=False),
        # the full layer of a ragged batch: the largest call
        dict(name="decode-batch-full", op="decode", dtype="bf16", batch=32, hq=64, hkv=8, dim=64, page=64, len_min=129,
             len_max=16384, window=0, sinks=0, logits=True, weigh=False),
        # the full layer of one long conversation, with the weights that an eviction goes by
        dict(name="decode-long-weights", op="decode", dtype="bf16", batch=1, hq=64, hkv=8, dim=64, page=64, len_min=131072,
             len_max=131072, window=0, sinks=0, logits=True, weigh=True),
        # large heads, a wide window, odd lengths, small pages
        dict(name="decode-wide-weights", op="decode", dtype="f16", batch=8, hq=32, hkv=4, dim=128, page=16, len_min=300,
             len_max=3000, window=1024, sinks=16, logits=False, weigh=True),
        # prompts cut down to a budget before decoding begins
        dict(name="evict-prompts", op="evict", dtype="bf16", batch=4, hkv=8, dim=64, page=64, len_min=16384, len_max=32768,
             keep=4096, trigger=4096, sinks=4, recent=128, steady=False),
        # a serving batch that goes over its budget a page at a time
        dict(name="evict-steps", op="evict", dtype="f16", batch=64, hkv=4, dim=128, page=32, len_min=1000, len_max=1088,
             keep=1024, trigger=1040, sinks=4, recent=64, steady=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "decode", "decode", "evict"])
    dtype = rng.choice(["bf16", "f16"])
    hq, hkv = rng.choice([(64, 8), (32, 4), (16, 16), (8, 1), (24, 8), (40, 2)])
    dim = rng.choice([16, 32, 64, 128])
    page = rng.choice([16, 32, 48, 64, 128])
    if op == "rotary":
        axes = rng.choice([1, 2, 3])
        rot = rng.choice([dim, dim // 2, dim - 4])
        batch = _log(rng, 1, 16)
        room = 67_000_000 // (batch * (hq + hkv) * dim)
        return dict(op=op, dtype=dtype, batch=batch, hq=hq, hkv=hkv, length=_log(rng, 1, max(1, min(16384, room))), dim=dim,
                    axes=axes, rot=rot, interleaved=rng.random() < 0.3, train=rng.random() < 0.5,
                    first=rng.choice([0, 0, 1 << 17, 1 << 20]))
    if op == "append":
        batch = _log(rng, 1, 256)
        most = 1 if rng.random() < 0.5 else _log(rng, 2, max(2, min(4096, 24000 // batch)))
        old = _log(rng, 1, 2000)
        return dict(op=op, dtype=dtype, batch=batch, hq=hq, hkv=hkv, dim=dim, page=page, new_min=1 if most == 1 else rng.randint(0, most),
                    new_max=most, old_min=rng.randint(0, old), old_max=old, axes=rng.choice([1, 3]), track=rng.random() < 0.5)
    if op == "decode":
        batch = _log(rng, 1, 256)
        longest = _log(rng, 1, max(1, min(131072, 16_000_000 // (batch * hkv * dim) * 8)))
        window = rng.choice([0, 0, 128, 1024])
        return dict(op=op, dtype=dtype, batch=batch, hq=hq, hkv=hkv, dim=dim, page=page, len_min=rng.randint(0, longest), len_max=longest,
                    window=window, sinks=rng.choice([0, 4, 16]) if window else 0, logits=rng.random() < 0.5,
                    weigh=rng.random() < 0.4)
    batch = _log(rng, 1, 64)
    longest = _log(rng, 64, max(64, min(65536, 8_000_000 // (batch * hkv * dim) * 8)))
    keep = rng.randint(32, longest)
    return dict(op=op, dtype=dtype, batch=batch, hkv=hkv, dim=dim, page=page, len_min=rng.randint(1, longest), len_max=longest,
                keep=keep, trigger=keep + rng.choice([0, 0, 16]), sinks=rng.choice([0, 4]),
                recent=rng.choice([0, 16, keep - 4]), steady=rng.random() < 0.5)


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, evenly spaced: known without a seed, so that the work is known too."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _visible(case):
    """Keys that the new token of each sequence sees."""
    seen = []
    for n in _spread(case["batch"], case["len_min"], case["len_max"]):
        w = case["window"] or n
        seen.append(min(n, w) + max(0, min(case["sinks"], n - w)))
    return seen


def _evicted(case):
    return [n for n in _spread(case["batch"], case["len_min"], case["len_max"]) if n > max(case["trigger"], case["keep"])]


def work(case):
    d, b = case["dim"], case["batch"]
    if case["op"] == "rotary":
        values = b * case["length"] * (case["hq"] + case["hkv"]) * d
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * 2 * values + 8 * case["axes"] * b * case["length"]),
                "flops": passes * 3 * b * case["length"] * (case["hq"] + case["hkv"]) * case["rot"]}
    if case["op"] == "append":
        t = sum(_spread(b, case["new_min"], case["new_max"]))
        return {"bytes": t * (2 * 2 * (case["hq"] + 2 * case["hkv"]) * d + 8 * case["axes"] + (8 * case["hkv"] if case["track"] else 0)),
                "flops": 3 * t * (case["hq"] + case["hkv"]) * d}
    if case["op"] == "decode":
        keys = sum(_visible(case))
        slots = sum(_spread(b, case["len_min"], case["len_max"]))
        return {"bytes": keys * case["hkv"] * d * 4 + 4 * b * case["hq"] * d + (8 * case["hkv"] * slots if case["weigh"] else 0),
                "flops": 4 * keys * case["hq"] * d}
    # an evicted entry in the kept part, or a kept one behind it, moves; the shares go by chance
    moved = sum(case["keep"] * (n - case["keep"]) // n for n in _evicted(case))
    slots = sum(_evicted(case))
    return {"bytes": case["hkv"] * (8 * slots + moved * (2 * 4 * d + 16)) + 8 * b, "flops": 0}


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, dtype, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(0.5).to(dtype)


def _order(g, n):
    return torch.randperm(n, generator=g, device="cuda")


def _positions(case, g, t):
    """[axes, t]: text counts up on every axis; pictures hold the time and walk over a grid."""
    pos = torch.arange(t, device="cuda").repeat(case["axes"], 1) + case.get("first", 0)
    if case["axes"] > 1:
        side = 24
        picture = (torch.arange(t, device="cuda") // (side * side)) % 2 == 0
        start = torch.randint(0, 4096, (1,), generator=g, device="cuda") + case.get("first", 0)
        cell = torch.arange(t, device="cuda") % (side * side)
        grid = [start + 0 * cell, start + cell // side, start + cell % side]
        pos = torch.stack([torch.where(picture, grid[a], pos[a]) for a in range(case["axes"])])
    return pos


def _sections(case, rot):
    n = rot // 2
    return {1: (n,), 2: (n // 2, n - n // 2), 3: (n - 2 * (3 * n // 8), 3 * n // 8, 3 * n // 8)}[case["axes"]]


def _rotation(case, s, rot):
    """The table of inverse frequencies and the axis that each goes by."""
    n = rot // 2
    s["inv_freq"] = (150000.0 ** (-torch.arange(n, device="cuda", dtype=torch.float64) / max(1, n))).float()
    s["sections"] = _sections(case, rot)
    s["axis"] = torch.repeat_interleave(torch.arange(case["axes"]), torch.tensor(s["sections"])).to("cuda")
    s["interleaved"], s["scale"] = case.get("interleaved", False), 1.25
    if own:
        s["rotary"] = _pkg("rotary").Rotary(s["inv_freq"], sections=s["sections"], interleaved=s["interleaved"], scale=s["scale"])


def _cache(case, s, g, lens, longest, shuffle=True):
    """Pages of a pool in random order, page tables that hold -1 behind each sequence, its lengths."""
    dtype, p, b, hkv, d = DTYPES[case["dtype"]], case["page"], case["batch"], case["hkv"], case["dim"]
    m = max(1, -(-longest // p))
    lens = torch.tensor(lens, device="cuda", dtype=torch.int32)
    order = _order(g, b) if shuffle else torch.arange(b, device="cuda")
    lens = lens[order]
    s["lens"], s["order"], s["page"] = lens, order, p
    n = b * m + 3
    table = _order(g, n)[: b * m].reshape(b, m).to(torch.int32)
    s["table"] = torch.where(torch.arange(m, device="cuda") * p < lens[:, None], table, -1)
    s["k"], s["v"] = _randn(g, dtype, n, hkv, p, d), _randn(g, dtype, n, hkv, p, d)


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": dict(case)}
    dtype, b, d = DTYPES[case["dtype"]], case["batch"], case["dim"]
    if case["op"] == "rotary":
        s["q"], s["kk"] = (_randn(g, dtype, b, h, case["length"], d) for h in (case["hq"], case["hkv"]))
        s["pos"] = torch.stack([_positions(case, g, case["length"]) for _ in range(b)], 1)
        if case["train"]:
            s["dq"], s["dk"] = (_randn(g, dtype, b, h, case["length"], d) for h in (case["hq"], case["hkv"]))
            s["q"].requires_grad_(), s["kk"].requires_grad_()
        _rotation(case, s, case["rot"])
        return s
    if case["op"] == "append":
        new, old = _spread(b, case["new_min"], case["new_max"]), _spread(b, case["old_min"], case["old_max"])
        _cache(case, s, g, [x + y for x, y in zip(new, old)], case["new_max"] + case["old_max"])
        new = torch.tensor(new, device="cuda", dtype=torch.int32)[s["order"]]
        s["cu"] = torch.nn.functional.pad(new.cumsum(0), (1, 0)).to(torch.int32)
        t = sum(_spread(b, case["new_min"], case["new_max"]))
        s["q"], s["new_k"], s["new_v"] = (_randn(g, dtype, t, h, d) for h in (case["hq"], case["hkv"], case["hkv"]))
        s["pos"] = _positions(case, g, t)
        _rotation(case, s, d)
        cap = s["table"].shape[1] * case["page"]
        if case["track"]:
            s["weights"] = torch.rand(b, case["hkv"], cap, generator=g, device="cuda")
            s["positions"] = torch.arange(cap, device="cuda", dtype=torch.int32).expand(b, case["hkv"], cap).contiguous()
            s["seen"] = s["lens"] + 100
        if own:
            s["cache"] = _pkg("paged").PagedKVCache(s["k"], s["v"], s["table"], s["lens"], weights=s.get("weights"),
                                                    positions=s.get("positions"), seen=s.get("seen"))
        return s
    _cache(case, s, g, _spread(b, case["len_min"], case["len_max"]), case["len_max"])
    cap = s["table"].shape[1] * case["page"]
    if case["op"] == "decode":
        # a token's query looks at some keys much harder than at others
        s["q"] = _randn(g, dtype, b, case["hq"], d) * 8
        s["logits"] = torch.randn(case["hq"], generator=g, device="cuda") if case["logits"] else None
        if case["weigh"]:
            s["weights"] = torch.rand(b, case["hkv"], cap, generator=g, device="cuda")
            s["new_weights"] = torch.zeros_like(s["weights"])
        if own:
            s["cache"] = _pkg("paged").PagedKVCache(s["k"], s["v"], s["table"], s["lens"], weights=s.get("weights"))
        return s
    # weights as attention leaves them: few large, most small, some never looked at
    h = case["hkv"]
    weights = torch.randn(b, h, cap, generator=g, device="cuda").mul_(2.5).exp_().mul_(1e-3)
    weights[torch.rand(b, h, cap, generator=g, device="cuda") < 0.05] = 0.0
    positions = torch.arange(cap, device="cuda", dtype=torch.int32).expand(b, h, cap)
    seen = s["lens"].clone()
    if case["steady"]:  # after earlier evictions: later tokens have gone into earlier places
        key = torch.rand(b, h, cap, generator=g, device="cuda") + 2.0 * (positions >= s["lens"][:, None, None])
        positions = key.argsort(-1).to(torch.int32)
        positions = torch.where(positions >= case["sinks"], positions + 500, positions)
        seen = seen + 500
    s["seen"] = seen
    # what a pass changes besides the places that it fills, as one buffer that the next pass takes anew: the pages need
    # no renewal, since the rows that are moved stay where they were, behind the kept part
    s["kept"] = torch.cat([s["lens"], weights.reshape(-1).view(torch.int32), positions.reshape(-1)])
    s["book"] = s["kept"].clone()
    s["lens"] = s["book"][:b]
    s["weights"] = s["book"][b: b + weights.numel()].view(torch.float32).view(b, h, cap)
    s["positions"] = s["book"][b + weights.numel():].view(b, h, cap)
    if own:
        s["cache"] = _pkg("paged").PagedKVCache(s["k"], s["v"], s["table"], s["lens"], weights=s["weights"],
                                                positions=s["positions"], seen=s["seen"])
    return s


# ---------------------------------------------------------------------------------------
# the operators' plain forms
# ---------------------------------------------------------------------------------------

def _angles(s, pos):
    """cos and sin, [..., n], of positions [axes, ...]; the angle in 64 bits, where far positions keep it."""
    a = pos[s["axis"]].double().movedim(0, -1) * s["inv_freq"].double()
    return (a.cos() * s["scale"]).float(), (a.sin() * s["scale"]).float()


def _rotate(s, x, cos, sin, inverse=False):
    """x [..., D] rotated by angles [..., n]: the first 2n values of a head turn, the others stay."""
    n = cos.shape[-1]
    y = x.float()
    turn = y[..., : 2 * n]
    if s["interleaved"]:
        u, w = turn[..., 0::2], turn[..., 1::2]
    else:
        u, w = turn[..., :n], turn[..., n:]
    if inverse:
        sin = -sin
    first, second = u * cos - w * sin, w * cos + u * sin
    turned = torch.stack([first, second], -1).flatten(-2) if s["interleaved"] else torch.cat([first, second], -1)
    return torch.cat([turned, y[..., 2 * n:]], -1).to(x.dtype)


def _rows(s, x, slots):
    """The rows [B, n, Hkv, D] of pages x at slots [B, n] of each sequence."""
    page = torch.gather(s["table"].long(), 1, slots // s["page"]).clamp_min(0)
    return x[page, :, slots % s["page"]]


def _rotary_run(s):
    if own:
        rot, train = _pkg("rotary"), s["case"]["train"]
        q, k = rot.apply_rotary(s["q"], s["kk"], s["pos"], s["rotary"])
        if not train:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["kk"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    with torch.no_grad():
        cos, sin = (x[:, None] for x in _angles(s, s["pos"]))
        out = {"q": _rotate(s, s["q"], cos, sin), "k": _rotate(s, s["kk"], cos, sin)}
        if s["case"]["train"]:
            out |= {"dq": _rotate(s, s["dq"], cos, sin, True), "dk": _rotate(s, s["dk"], cos, sin, True)}
    return out


def _append_run(s):
    c = s["case"]
    out = {"k": s["k"], "v": s["v"]}
    if c["track"]:
        out |= {"weights": s["weights"], "positions": s["positions"]}
    if own:
        cu = None if c["new_max"] == 1 and c["new_min"] == 1 else s["cu"]
        out["q"] = s["cache"].append(s["new_k"], s["new_v"], cu_new=cu, q=s["q"], positions=s["pos"], rotary=s["rotary"])
        return out
    cos, sin = (x[:, None] for x in _angles(s, s["pos"]))
    out["q"] = _rotate(s, s["q"], cos, sin)
    t = s["q"].shape[0]
    token = torch.arange(t, device=s["q"].device)
    seq = torch.searchsorted(s["cu"][1:].contiguous(), token.to(torch.int32), right=True)
    back = (s["cu"][1:][seq] - token).long()  # how far from its sequence's end the token is
    slot = s["lens"][seq].long() - back
    page = s["table"][seq, slot // s["page"]].long()
    s["k"][page, :, slot % s["page"]] = _rotate(s, s["new_k"], cos, sin)
    s["v"][page, :, slot % s["page"]] = s["new_v"]
    if c["track"]:
        s["weights"][seq, :, slot] = 0.0
        s["positions"][seq, :, slot] = (s["seen"][seq].long() - back).to(torch.int32)[:, None].expand(-1, c["hkv"])
    return out


def _decode_run(s):
    c = s["case"]
    scale = 1.0 / math.sqrt(c["dim"])
    if own:
        o = s["cache"].decode(s["q"], window_size=c["window"] or None, sink_size=c["sinks"], softmax_scale=scale,
                              sinks=s["logits"], weights_out=s.get("new_weights"))
        return {"o": o, "weights": s["new_weights"]} if c["weigh"] else {"o": o}
    b, hkv, d, cap = c["batch"], c["hkv"], c["dim"], s["table"].shape[1] * s["page"]
    n = s["lens"].long()[:, None]
    first = (n - (c["window"] or cap)).clamp_min(0)  # the window's first slot
    far = first.clamp_max(c["sinks"])                # sink slots before it
    at = torch.arange(min(cap, c["window"] + c["sinks"]) if c["window"] else cap, device=n.device)[None]
    slots = torch.where(at < far, at, at + first - far)
    ok = slots < n
    slots = torch.where(ok, slots, 0)
    q = s["q"].float().view(b, hkv, -1, d)
    k, v = (_rows(s, x, slots).float().transpose(1, 2) for x in (s["k"], s["v"]))
    score = (q @ k.transpose(-1, -2)) * scale
    score = torch.where(ok[:, None, None], score, -torch.inf)
    most = score.amax(-1, keepdim=True)
    if s["logits"] is not None:
        sink = s["logits"].view(1, hkv, -1, 1)
        most = torch.maximum(most, sink)
    most = torch.where(most == -torch.inf, 0.0, most)
    e = torch.exp(score - most)
    total = e.sum(-1, keepdim=True)
    if s["logits"] is not None:
        total = total + torch.exp(sink - most)
    p = e / torch.where(total == 0, 1.0, total)
    o = (p @ v).reshape(b, -1, d).to(s["q"].dtype)
    if not c["weigh"]:
        return {"o": o}
    new = s["weights"].scatter_add(2, slots[:, None].expand(-1, hkv, -1), p.sum(2))
    live = (torch.arange(cap, device=n.device) < n)[:, None]
    return {"o": o, "weights": torch.where(live, new, s["new_weights"])}


def _evict_run(s):
    c = s["case"]
    s["book"].copy_(s["kept"])  # the lengths, weights and positions of before
    out = {"k": s["k"], "v": s["v"], "lens": s["lens"], "weights": s["weights"], "positions": s["positions"]}
    if own:
        s["cache"].evict(c["keep"], sink_size=c["sinks"], recent=c["recent"], trigger=c["trigger"])
        return out
    b, h, cap, keep = c["batch"], c["hkv"], s["weights"].shape[2], c["keep"]
    if keep >= cap:
        return out
    n = s["lens"].long()[:, None, None]
    slot = torch.arange(cap, device=n.device).expand(b, h, cap)
    held = (s["positions"] < c["sinks"]) | (s["positions"] >= (s["seen"] - c["recent"])[:, None, None])
    rank = torch.where(slot >= n, 0, torch.where(held, 2, 1))
    by = s["weights"].sort(dim=-1, descending=True, stable=True).indices
    by = by.gather(-1, rank.gather(-1, by).sort(dim=-1, descending=True, stable=True).indices)
    kept = torch.zeros(b, h, cap, dtype=torch.bool, device=n.device).scatter_(-1, by[..., :keep], True)
    kept = torch.where(n > max(c["trigger"], keep), kept, slot < n)
    hole = ~kept & (slot < keep) & (slot < n)
    mover = kept & (slot >= keep) & (n > max(c["trigger"], keep))
    # the i-th place that came free, from the front, takes the i-th kept entry behind the budget
    source = (~mover).to(torch.int8).sort(dim=-1, stable=True).indices
    nth = (hole.cumsum(-1) - 1).clamp_min(0)
    src = torch.where(hole, source.gather(-1, nth), slot)[..., :keep]
    dst = slot[..., :keep]
    head = torch.arange(h, device=n.device)[None, :, None]
    table = s["table"].long().clamp_min(0)[:, None].expand(b, h, -1)
    there, here = table.gather(-1, dst // s["page"]), table.gather(-1, src // s["page"])
    hole = hole[..., :keep]
    there, to, heads = there[hole], (dst % s["page"])[hole], head.expand(b, h, keep)[hole]
    here, at = here[hole], (src % s["page"])[hole]
    s["k"][there, heads, to] = s["k"][here, heads, at]
    s["v"][there, heads, to] = s["v"][here, heads, at]
    s["weights"][..., :keep] = s["weights"].gather(-1, src)
    s["positions"][..., :keep] = s["positions"].gather(-1, src)
    s["lens"].copy_(torch.where(s["lens"] > max(c["trigger"], keep), keep, s["lens"]))
    return out


def run(state):
    return {"rotary": _rotary_run, "append": _append_run, "decode": _decode_run, "evict": _evict_run}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------
# the operators' definitions in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------------------

def _exact_turn(s, x, pos, inverse=False):
    """x [..., t, D] with the matrix of each position: pair i of a head as a complex number times exp(i angle)."""
    inv, n = s["inv_freq"].double(), s["inv_freq"].numel()
    angle = torch.stack([pos[int(s["axis"][i])].double() * inv[i] for i in range(n)], -1)
    unit = torch.polar(torch.full_like(angle, s["scale"]), -angle if inverse else angle)
    y = x.detach().double().clone()
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if s["interleaved"] else (slice(0, n), slice(n, 2 * n))
    z = torch.complex(y[..., a], y[..., b]) * unit
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _exact_slots(s, b, slots):
    return s["table"][b, slots // s["page"]].long(), slots % s["page"]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        turn = lambda x, inv: torch.stack([_exact_turn(s, x[i], s["pos"][:, i], inv) for i in range(x.shape[0])])  # noqa: E731
        out = {"q": turn(s["q"], False), "k": turn(s["kk"], False)}
        if case["train"]:
            out |= {"dq": turn(s["dq"], True), "dk": turn(s["dk"], True)}
        return out
    if case["op"] == "append":
        out = {"k": s["k"].double(), "v": s["v"].double(), "q": _exact_turn(s, s["q"].transpose(0, 1), s["pos"]).transpose(0, 1)}
        turned = _exact_turn(s, s["new_k"].transpose(0, 1), s["pos"]).transpose(0, 1)
        cu, lens = s["cu"].tolist(), s["lens"].tolist()
        if case["track"]:
            out |= {"weights": s["weights"].double(), "positions": None}
        for b in range(case["batch"]):
            lo, hi = cu[b], cu[b + 1]
            slots = torch.arange(lens[b] - (hi - lo), lens[b], device="cuda")
            page, row = _exact_slots(s, b, slots)
            out["k"][page, :, row], out["v"][page, :, row] = turned[lo:hi], s["new_v"][lo:hi].double()
            if case["track"]:
                out["weights"][b, :, slots] = 0.0
        return out
    if case["op"] == "decode":
        heads = case["hq"] // case["hkv"]
        o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        weights = s["new_weights"].double() if case["weigh"] else None
        for b, n in enumerate(s["lens"].tolist()):
            if n == 0:
                continue
            slots = torch.arange(n, device="cuda")
            seen = torch.ones_like(slots, dtype=torch.bool)
            if case["window"]:
                seen = (n - 1 - slots < case["window"]) | (slots < case["sinks"])
            vis = slots[seen]
            page, row = _exact_slots(s, b, vis)
            k, v = s["k"][page, :, row].double(), s["v"][page, :, row].double()
            q = s["q"][b].double().view(case["hkv"], heads, -1)
            score = torch.einsum("hgd,nhd->hgn", q, k) / math.sqrt(case["dim"])
            if case["logits"]:
                p = torch.softmax(torch.cat([score, s["logits"].double().view(case["hkv"], heads, 1)], -1), -1)[..., :-1]
            else:
                p = torch.softmax(score, -1)
            o[b] = torch.einsum("hgn,nhd->hgd", p, v).reshape(case["hq"], -1)
            if case["weigh"]:
                weights[b, :, :n] = s["weights"][b, :, :n].double()
                weights[b, :, vis] += p.sum(1)
        return {"o": o, "weights": weights} if case["weigh"] else {"o": o}
    k, v, w = s["k"].double(), s["v"].double(), s["weights"].double()
    out = {"k": k, "v": v, "lens": None, "weights": w, "positions": None}
    keep = case["keep"]
    for b, n in enumerate(s["lens"].tolist()):
        if n <= max(case["trigger"], keep):
            continue
        for h in range(case["hkv"]):
            pos = s["positions"][b, h, :n]
            held = (pos < case["sinks"]) | (pos >= int(s["seen"][b]) - case["recent"])
            value = torch.where(held, torch.inf, w[b, h, :n])
            chosen = torch.argsort(-value, stable=True)[:keep]
            kept = torch.zeros(n, dtype=torch.bool, device="cuda")
            kept[chosen] = True
            dst = torch.nonzero(~kept[:keep])[:, 0]
            src = torch.nonzero(kept[keep:])[:, 0] + keep
            (pd, rd), (ps, rs) = _exact_slots(s, b, dst), _exact_slots(s, b, src)
            k[pd, h, rd], v[pd, h, rd] = s["k"][ps, h, rs].double(), s["v"][ps, h, rs].double()
            w[b, h, dst] = w[b, h, src]
    return out
