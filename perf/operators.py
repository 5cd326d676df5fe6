"""Cases of the selection operators for language models: routing to experts, beam selection with
the reordering of states, and eviction from a key/value cache.

Each case is one call as a serving or training program makes it, on tensors that such a program
holds on the GPU.  `run` computes it either in plain torch operations or, with `own` set, through
this repository's binding.  The selections compare scores in 64 bits, since two scores next to
each other decide which index comes out; everything else is in 32 bits and rounded once.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
NEG = float("-inf")


# ------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of a small serving batch: latency counts; lists by expert for the products
        {"name": "route step 64x256", "op": "route", "tokens": 64, "experts": 256, "k": 8, "type": "bf16",
         "score": "sigmoid", "renormalise": True, "scale": 2.5, "bias": True, "groups": 8,
         "groups_kept": 4, "group_top": 2, "padded": 0.0},
        # a padded batch of prompts through a router of an odd number of experts
        {"name": "route prompt 4999x60", "op": "route", "tokens": 4999, "experts": 60, "k": 4, "type": "fp16",
         "score": "softmax", "renormalise": False, "scale": 1.0, "bias": False, "groups": 1,
         "groups_kept": 1, "group_top": 1, "padded": 0.1},
        # a training or prefill batch with grouped routing and a balance bias, logits in 32 bits
        {"name": "route batch 16384x256", "op": "route", "tokens": 16384, "experts": 256, "k": 8, "type": "fp32",
         "score": "sigmoid", "renormalise": True, "scale": 2.5, "bias": True, "groups": 8,
         "groups_kept": 4, "group_top": 2, "padded": 0.0},
        # the router's backward pass in a small step
        {"name": "route grad 777x256", "op": "route_grad", "tokens": 777, "experts": 256, "k": 8, "type": "fp32",
         "score": "sigmoid", "renormalise": True, "scale": 2.5},
        # the router's backward pass of a large batch, through the whole softmax
        {"name": "route grad 32768x128", "op": "route_grad", "tokens": 32768, "experts": 128, "k": 6, "type": "bf16",
         "score": "softmax", "renormalise": False, "scale": 1.0},
        # one sequence searched with four beams
        {"name": "beam 1x4x32000", "op": "beam", "batch": 1, "beams": 4, "vocab": 32000, "k": 8, "type": "bf16",
         "finished": False},
        # an odd vocabulary, logits in 32 bits, some beams finished
        {"name": "beam 16x5x50001", "op": "beam", "batch": 16, "beams": 5, "vocab": 50001, "k": 5, "type": "fp32",
         "finished": True},
        # a full serving batch with a large vocabulary
        {"name": "beam 64x8x128000", "op": "beam", "batch": 64, "beams": 8, "vocab": 128000, "k": 16, "type": "bf16",
         "finished": False},
        # the caches of a small model follow four beams
        {"name": "reorder 8x1x4", "op": "reorder", "outer": 8, "batch": 1, "beams": 4, "segments": 8,
         "rows": 64, "used": 50, "dim": 64},
        # the caches of 24 layers (keys and values) follow the beams of a batch
        {"name": "reorder 48x8x4", "op": "reorder", "outer": 48, "batch": 8, "beams": 4, "segments": 8,
         "rows": 512, "used": 411, "dim": 64},
        # a decode step at the cache's budget: one entry leaves each head's cache
        {"name": "evict step 32x8x4097", "op": "evict", "batch": 32, "heads": 8, "group": 4, "queries": 1,
         "capacity": 4160, "length": 4097, "ragged": False, "budget": 4096, "recent": 256, "sink": 4, "dim": 64,
         "type": "bf16"},
        # prompts of different lengths are cut to the budget by the weights of their last queries
        {"name": "evict prompt 4x8x16384", "op": "evict", "batch": 4, "heads": 8, "group": 4, "queries": 16,
         "capacity": 16384, "length": 16384, "ragged": True, "budget": 1024, "recent": 64, "sink": 4, "dim": 128,
         "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "route_grad", "beam", "reorder", "evict"])
    kind = rng.choice(["fp32", "fp16", "bf16"])
    if op in ("route", "route_grad"):
        grouped = op == "route" and rng.random() < 0.5
        groups = rng.choice([2, 4, 8]) if grouped else 1
        experts = groups * _log(rng, 8, 256 // groups) if grouped else _log(rng, 8, 256)
        kept = rng.randint(1, groups)
        k = rng.randint(1, min(8, experts // groups * kept))
        c = {"op": op, "tokens": _log(rng, 1, 16384), "experts": experts, "k": k, "type": kind,
             "score": rng.choice(["softmax", "sigmoid"]), "renormalise": rng.random() < 0.5,
             "scale": round(rng.uniform(0.5, 3.0), 2)}
        if op == "route":
            c.update(bias=rng.random() < 0.5, groups=groups, groups_kept=kept,
                     group_top=rng.choice([1, 2]) if grouped else 1, padded=rng.choice([0.0, 0.1, 0.5]))
        return c
    if op == "beam":
        beams, vocab = rng.randint(1, 8), _log(rng, 1000, 128000)
        return {"op": op, "batch": _log(rng, 1, min(64, 30_000_000 // (beams * vocab))), "beams": beams,
                "vocab": vocab, "k": rng.randint(1, 2 * beams), "type": kind, "finished": rng.random() < 0.5}
    if op == "reorder":
        rows = _log(rng, 16, 512)
        return {"op": op, "outer": rng.randint(1, 48), "batch": rng.randint(1, 8), "beams": rng.randint(2, 4),
                "segments": rng.choice([1, 2, 8]), "rows": rows, "used": rng.randint(1, rows),
                "dim": rng.choice([20, 64, 128]) if rows <= 256 else 64}
    length = _log(rng, 64, 8192)
    return {"op": op, "batch": rng.randint(1, 8), "heads": rng.choice([1, 2, 4, 8]), "group": rng.choice([1, 2, 4]),
            "queries": rng.choice([1, 1, 2, 8]), "capacity": length + rng.randint(0, 64), "length": length,
            "ragged": rng.random() < 0.5, "budget": rng.randint(length // 8 + 1, length), "recent": rng.randint(0, length // 16),
            "sink": rng.choice([0, 1, 4]), "dim": rng.choice([40, 64, 128]), "type": kind}


# ------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    s = {"case": case}
    if case["op"] in ("route", "route_grad"):
        t, e, k = case["tokens"], case["experts"], case["k"]
        # some experts are liked more than others, as in a trained router
        s["logits"] = (1.5 * normal(t, e) + 0.5 * normal(e)).to(TYPES[case["type"]])
        if case["op"] == "route":
            s["bias"] = 0.05 * normal(e) if case["bias"] else None
            s["mask"] = (uniform(t) >= case["padded"]).to(torch.uint8) if case["padded"] else None
        else:
            s["ids"] = torch.topk(s["logits"].float(), k, dim=-1).indices.to(torch.int32)
            s["grad"] = normal(t, k)
    elif case["op"] == "beam":
        b, w, v = case["batch"], case["beams"], case["vocab"]
        x = torch.empty(b, w, v, device="cuda", dtype=TYPES[case["type"]])
        for i in range(b):  # a few likely tokens in front of a broad rest
            x[i] = (2.0 * normal(w, v) + 6.0 * (uniform(w, v) < 2e-4) * uniform(w, v)).to(x.dtype)
        s["logits"] = x
        s["cum"] = torch.sort(-10.0 * uniform(b, w), dim=-1, descending=True).values
        s["finished"] = (uniform(b, w) < 0.2).to(torch.uint8) if case["finished"] else None
        s["eos"] = 2
    elif case["op"] == "reorder":
        o, b, w = case["outer"], case["batch"], case["beams"]
        s["states"] = torch.empty(o, b, w, case["segments"], case["rows"], case["dim"], device="cuda", dtype=torch.bfloat16)
        s["states"].normal_(generator=g)
        s["parents"] = torch.randint(0, w, (b, w), device="cuda", generator=g, dtype=torch.int32)
    else:
        b, h, q, c, n = case["batch"], case["heads"], case["queries"], case["capacity"], case["length"]
        lens = torch.full((b,), n, device="cuda", dtype=torch.int32)
        if case["ragged"]:
            lens = (n // 2 + 1 + (uniform(b) * (n - n // 2)).int()).clamp(max=n)
        s["lens"] = lens
        slot = torch.arange(c, device="cuda")
        live = slot < lens[:, None]
        logits = 2.0 * normal(b, h * case["group"], q, c)
        logits.masked_fill_(~live[:, None, None, :], NEG)
        s["weights"] = torch.softmax(logits, -1).to(TYPES[case["type"]])
        s["acc"] = -torch.log1p(-uniform(b, h, c)) * (4.0 / n)
        # earlier evictions have moved entries about: positions are not in the slots' order
        order = torch.argsort(uniform(b, h, c) + (~live[:, None, :]).float() * 2, dim=-1)
        s["pos"] = (order * 2 if case["queries"] == 1 else slot.expand(b, h, c)).to(torch.int32).contiguous()
        s["seen"] = (lens * (2 if case["queries"] == 1 else 1)).to(torch.int32)
        for name in ("keys", "values"):
            s[name] = torch.empty(b, h, c, case["dim"], device="cuda", dtype=torch.bfloat16)
            s[name].normal_(generator=g)
    return s


# ------------------------------------------------------------------------- the plain forms
def _route_scores(x, score):
    """Scores in 64 bits; logits of -inf or NaN are no choice and weigh nothing."""
    x = x.double()
    x = torch.where(torch.isnan(x), NEG, x)
    if score == "sigmoid":
        return x, torch.sigmoid(x)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(torch.where(x == m, 0.0, x - m))
    e = torch.where(x == NEG, 0.0, e)
    total = e.sum(-1, keepdim=True)
    return x, e / torch.where(total == 0, 1.0, total)


def _route(s):
    c = s["case"]
    t, n, k = c["tokens"], c["experts"], c["k"]
    x, p = _route_scores(s["logits"], c["score"])
    sums = p if s["bias"] is None else p + s["bias"].double()
    key = x if s["bias"] is None else torch.where(x == NEG, NEG, sums)
    if c["groups"] > 1:
        per = (key if s["bias"] is None and c["group_top"] == 1 else torch.where(key == NEG, NEG, sums)).view(t, c["groups"], -1)
        top = torch.sort(per, dim=-1, descending=True).values[..., :c["group_top"]]
        rank = torch.where(top[..., 0] == NEG, NEG, torch.where(top == NEG, 0.0, top).sum(-1))
        best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :c["groups_kept"]]
        kept = torch.zeros(t, c["groups"], dtype=torch.bool, device=x.device).scatter_(1, best, True)
        key = torch.where(kept[..., None], key.view(t, c["groups"], -1), NEG).view(t, n)
    if s["mask"] is not None:
        key = torch.where(s["mask"][:, None] != 0, key, NEG)
    order = torch.sort(key, dim=-1, descending=True, stable=True)
    ids = torch.where(order.values[:, :k] == NEG, -1, order.indices[:, :k])
    w = torch.where(ids < 0, 0.0, p.gather(1, ids.clamp(min=0)))
    if c["renormalise"]:
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total == 0, 1.0, total)
    flat = ids.reshape(-1)
    by = torch.sort(torch.where(flat < 0, n, flat), stable=True)
    start = torch.searchsorted(by.values, torch.arange(n + 1, device=x.device)).to(torch.int32)
    slots = torch.where(by.values < n, by.indices, -1).to(torch.int32)
    return {"ids": ids.to(torch.int32), "weights": (c["scale"] * w).float(), "start": start, "slots": slots}


def _route_grad(s):
    c = s["case"]
    ids, g, x = s["ids"].long(), s["grad"], s["logits"].float()
    if c["score"] == "softmax":
        p = torch.softmax(x, -1)
    else:
        p = torch.sigmoid(x)
    chosen = p.gather(1, ids)
    if c["renormalise"]:
        w = chosen / chosen.sum(-1, keepdim=True)
        d = w * (g - (g * w).sum(-1, keepdim=True))
        if c["score"] == "sigmoid":
            d = d * torch.sigmoid(-x.gather(1, ids))
        out = torch.zeros_like(x).scatter_add_(1, ids, d)
    elif c["score"] == "softmax":
        wide = torch.zeros_like(x).scatter_add_(1, ids, g)
        out = p * (wide - (g * chosen).sum(-1, keepdim=True))
    else:
        out = torch.zeros_like(x).scatter_add_(1, ids, g * chosen * torch.sigmoid(-x.gather(1, ids)))
    return (c["scale"] * out).to(s["logits"].dtype)


def _beam(s):
    c = s["case"]
    b, w, v, k = c["batch"], c["beams"], c["vocab"], c["k"]
    x = s["logits"].float()
    x = torch.where(torch.isnan(x), NEG, x)
    m = x.amax(-1, keepdim=True)
    # the order of two beams' candidates hangs on the sums over the vocabulary: 64 bits
    total = torch.exp(torch.where(x == m, 0.0, x.double() - m)).sum(-1, keepdim=True)
    # each beam's best tokens by one whole number: the logit's order, then the lower token
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    order = (order << 32) | (v - 1 - torch.arange(v, device=x.device))
    tokens = v - 1 - (torch.topk(order, min(k, v), dim=-1).values & 0xFFFFFFFF)
    best = x.gather(-1, tokens)
    cum = s["cum"].double()[..., None]
    key = cum + (torch.where(best == m, 0.0, best.double() - m) - torch.log(total))
    key = torch.where((best == NEG) | ~torch.isfinite(cum), NEG, key)
    if s["finished"] is not None:
        done = s["finished"][..., None] != 0
        first = torch.arange(key.shape[-1], device=x.device) == 0
        key = torch.where(done, torch.where(first & torch.isfinite(cum), cum, NEG), key)
        tokens = torch.where(done, s["eos"], tokens)
    flat = key.view(b, -1)
    if flat.shape[1] < k:
        flat = torch.nn.functional.pad(flat, (0, k - flat.shape[1]), value=NEG)
    top = torch.sort(flat, dim=-1, descending=True, stable=True)
    score, at = top.values[:, :k], top.indices[:, :k]
    none = score == NEG
    at = torch.where(none, 0, at)
    parent = torch.where(none, -1, at // key.shape[-1])
    token = torch.where(none, -1, tokens.view(b, -1).gather(1, at))
    return {"parents": parent.to(torch.int32), "tokens": token.to(torch.int32), "scores": score.float()}


def _reorder(s):
    x, u = s["states"], s["case"]["used"]
    b, w = s["parents"].shape
    rows = (torch.arange(b, device=x.device)[:, None] * w + s["parents"]).view(-1)
    part = x.view(x.shape[0], b * w, *x.shape[3:])[:, :, :, :u]
    part.copy_(part[:, rows])
    return x


def _evict(s):
    c = s["case"]
    b, h, n, budget = c["batch"], c["heads"], c["capacity"], c["budget"]
    if "out" not in s:  # a program keeps two sets of these and swaps them
        s["out"] = torch.zeros_like(s["acc"]), torch.zeros_like(s["pos"])
    slot = torch.arange(n, device="cuda")
    lens = s["lens"].long()[:, None, None]
    live = (slot < lens).expand(b, h, n)
    w = s["weights"].view(b, h, c["group"] * c["queries"], n)
    acc = (s["acc"].double() + w.sum(2, dtype=torch.float64)).float()
    new = torch.clamp(s["lens"].long(), max=budget)[:, None, None]
    pos = s["pos"]
    fixed = (pos < c["sink"]) | (pos >= s["seen"][:, None, None] - c["recent"])
    key = torch.where(live, torch.where(fixed, math.inf, acc.double()), NEG)
    rank = torch.empty_like(slot).expand(b, h, n).contiguous()
    rank.scatter_(2, torch.sort(key, dim=-1, descending=True, stable=True).indices, slot.expand(b, h, n))
    keep = (rank < new) & live
    holes = (~keep & (slot < new)).nonzero(as_tuple=True)
    tails = (keep & (slot >= new)).nonzero(as_tuple=True)
    s["keys"][holes] = s["keys"][tails]
    s["values"][holes] = s["values"][tails]
    out_acc, out_pos = s["out"]
    acc[holes], moved = acc[tails], pos.clone()
    moved[holes] = pos[tails]
    torch.where(slot < new, acc, out_acc, out=out_acc)
    torch.where(slot < new, moved, out_pos, out=out_pos)
    return {"lens": new.view(-1).to(torch.int32), "acc": out_acc, "pos": out_pos, "keys": s["keys"], "values": s["values"]}


# ------------------------------------------------------------------------- the framework's calls
def _binding():
    at = os.path.join("metal-flat_b200", "python")
    if at not in sys.path:
        sys.path.insert(0, at)
    import mflat_b200
    return mflat_b200


def _make(s):
    """What a program keeps from call to call: the operator's handle, results, workspace."""
    M, c = _binding(), s["case"]

    def empty(*shape, dtype=torch.int32):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    if c["op"] == "route":
        t, n, k = c["tokens"], c["experts"], c["k"]
        op = M.Router(n, k, score=c["score"], dtype=c["type"], renormalise=c["renormalise"], scale=c["scale"],
                      groups=c["groups"], groups_kept=c["groups_kept"], group_top=c["group_top"])
        out = {"ids": empty(t, k), "weights": empty(t, k, dtype=torch.float32), "start": empty(n + 1),
               "slots": torch.full((t * k,), -1, device="cuda", dtype=torch.int32)}
        room = op.workspace_bytes(t)
    elif c["op"] == "route_grad":
        op = M.Router(c["experts"], c["k"], score=c["score"], dtype=c["type"], renormalise=c["renormalise"], scale=c["scale"])
        out, room = torch.empty_like(s["logits"]), 0
    elif c["op"] == "beam":
        op = M.BeamSearch(c["beams"], c["vocab"], c["k"], dtype=c["type"], eos=s["eos"])
        out = {"parents": empty(c["batch"], c["k"]), "tokens": empty(c["batch"], c["k"]),
               "scores": empty(c["batch"], c["k"], dtype=torch.float32)}
        room = op.workspace_bytes(c["batch"])
    elif c["op"] == "reorder":
        op, out, room = M.beam_reorder_device, s["states"], 0
    else:
        row = 2 * c["dim"]
        op = M.CacheEviction(c["heads"], c["group"], c["capacity"], c["budget"], key_bytes=row, value_bytes=row,
                             recent=c["recent"], sink=c["sink"], dtype=c["type"])
        out = {"lens": empty(c["batch"]), "acc": torch.zeros_like(s["acc"]), "pos": torch.zeros_like(s["pos"]),
               "keys": s["keys"], "values": s["values"]}
        room = op.workspace_bytes(c["batch"])
    s["op"], s["result"], s["room"] = op, out, empty(max(room, 1), dtype=torch.uint8)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _own(s):
    if "op" not in s:
        _make(s)
    c, op, out, room = s["case"], s["op"], s["result"], s["room"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "route":
        op.route_device(s["logits"].data_ptr(), c["tokens"], out["ids"].data_ptr(), out["weights"].data_ptr(),
                        bias=_ptr(s["bias"]), mask=_ptr(s["mask"]), start=out["start"].data_ptr(),
                        slots=out["slots"].data_ptr(), ws=room.data_ptr(), ws_bytes=room.numel(), stream=stream)
    elif c["op"] == "route_grad":
        op.backward_device(s["logits"].data_ptr(), c["tokens"], s["ids"].data_ptr(), s["grad"].data_ptr(),
                           out.data_ptr(), stream=stream)
    elif c["op"] == "beam":
        op.select_device(s["logits"].data_ptr(), s["cum"].data_ptr(), c["batch"], out["parents"].data_ptr(),
                         out["tokens"].data_ptr(), out["scores"].data_ptr(), finished=_ptr(s["finished"]),
                         ws=room.data_ptr(), ws_bytes=room.numel(), stream=stream)
    elif c["op"] == "reorder":
        line = 2 * c["dim"]
        op(out.data_ptr(), s["parents"].data_ptr(), c["outer"], c["batch"], c["beams"], c["used"] * line,
           segments=c["segments"], segment_stride=c["rows"] * line, stream=stream)
    else:
        op.evict_device(c["batch"], s["lens"].data_ptr(), s["seen"].data_ptr(), s["acc"].data_ptr(),
                        s["pos"].data_ptr(), s["keys"].data_ptr(), s["values"].data_ptr(), out["lens"].data_ptr(),
                        out_acc=out["acc"].data_ptr(), out_pos=out["pos"].data_ptr(), weights=s["weights"].data_ptr(),
                        queries=c["queries"], ws=room.data_ptr(), ws_bytes=room.numel(), stream=stream)
    return out


def run(state):
    if own:
        return _own(state)
    return {"route": _route, "route_grad": _route_grad, "beam": _beam, "reorder": _reorder,
            "evict": _evict}[state["case"]["op"]](state)


# ------------------------------------------------------------------------- what a pass cannot do without
def _moved(case):
    """Rows that an eviction moves in one head's cache, as expected: kept entries are spread evenly
    over the slots where positions are shuffled, and the recent ones are at the end otherwise."""
    n, m = case["length"] * (0.75 if case["ragged"] else 1.0), case["budget"]
    if n <= m:
        return 0.0
    return max(m * (n - m) / n, min(case["recent"], n - m) if case["queries"] > 1 else 0.0)


def work(case):
    if case["op"] in ("route", "route_grad"):
        t, e, k, z = case["tokens"], case["experts"], case["k"], SIZE[case["type"]]
        if case["op"] == "route":
            return {"bytes": t * e * z + t * k * 12 + (e + 1) * 4 + (e * 4 if case["bias"] else 0) + (t if case["padded"] else 0),
                    "flops": t * e * 8}
        whole = case["score"] == "softmax" and not case["renormalise"]
        return {"bytes": t * e * z + t * k * 8 + t * (e if whole else k) * z, "flops": t * e * 6 if whole else t * k * 12}
    if case["op"] == "beam":
        n = case["batch"] * case["beams"]
        return {"bytes": n * case["vocab"] * SIZE[case["type"]] * (0.8 if case["finished"] else 1) + n * 4 + case["batch"] * case["k"] * 12,
                "flops": n * case["vocab"] * 4}
    if case["op"] == "reorder":
        w = case["beams"]
        read, written = w * (1 - (1 - 1 / w) ** (w - 1)), w - 1
        return {"bytes": (read + written) * case["outer"] * case["batch"] * case["segments"] * case["used"] * case["dim"] * 2 + case["batch"] * w * 4,
                "flops": 0}
    heads = case["batch"] * case["heads"]
    n = case["length"] * (0.75 if case["ragged"] else 1.0)
    kept = min(n, case["budget"])
    return {"bytes": heads * (n * (case["group"] * case["queries"] * SIZE[case["type"]] + 8) + kept * 8 + _moved(case) * 8 * case["dim"]),
            "flops": heads * n * case["group"] * case["queries"]}


# ------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    """The operators' results from their definitions, in numpy's 64 bits, row by row."""
    s = prepare(case, seed)

    def host(name):
        t = s[name]
        return None if t is None else (t.double() if t.is_floating_point() else t).cpu().numpy()

    if case["op"] in ("route", "route_grad"):
        x, k = host("logits"), case["k"]
        if case["score"] == "sigmoid":
            p = 1.0 / (1.0 + np.exp(-x))
        else:
            p = np.exp(x - x.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
        if case["op"] == "route":
            bias, mask = host("bias"), host("mask")
            w = np.zeros((case["tokens"], k))
            size = case["experts"] // case["groups"]
            for t in range(case["tokens"]):
                if mask is not None and not mask[t]:
                    continue
                c = x[t] if bias is None else p[t] + bias
                open_ = np.arange(case["experts"])
                if case["groups"] > 1:
                    r = x[t] if bias is None and case["group_top"] == 1 else p[t] + (0 if bias is None else bias)
                    r = np.sort(r.reshape(-1, size), 1)[:, -case["group_top"]:].sum(1)
                    best = np.argsort(-r, kind="stable")[:case["groups_kept"]]
                    open_ = np.sort((best[:, None] * size + np.arange(size)).ravel())
                ids = open_[np.lexsort((open_, -c[open_]))[:k]]
                w[t] = p[t, ids] / (p[t, ids].sum() if case["renormalise"] else 1.0)
            return {"ids": None, "weights": torch.from_numpy(case["scale"] * w), "start": None, "slots": None}
        ids, g = host("ids"), host("grad")
        out = np.zeros_like(x)
        for t in range(case["tokens"]):
            # the weights' matrix of derivatives by the logits, [k][experts]
            i, j = ids[t], np.arange(len(ids[t]))
            if case["score"] == "softmax":
                d = -p[t, i, None] * p[t]
                d[j, i] += p[t, i]
            else:
                d = np.zeros((len(i), case["experts"]))
                d[j, i] = p[t, i] * (1 - p[t, i])
            if case["renormalise"]:
                total = p[t, i].sum()
                d = d / total - p[t, i, None] * d.sum(0) / total ** 2
            out[t] = case["scale"] * (g[t] @ d)
        return torch.from_numpy(out)
    if case["op"] == "beam":
        cum, done = host("cum"), host("finished")
        scores = np.full((case["batch"], case["k"]), NEG)
        for b in range(case["batch"]):
            x = s["logits"][b].double().cpu().numpy()
            key = cum[b][:, None] + x - np.logaddexp.reduce(x.astype(np.longdouble), 1)[:, None].astype(np.float64) \
                if x.size < 300_000 else cum[b][:, None] + x - (x.max(1) + np.log(np.exp(x - x.max(1, keepdims=True)).sum(1)))[:, None]
            if done is not None:
                key[done[b] != 0] = NEG
                key[done[b] != 0, s["eos"]] = cum[b][done[b] != 0]
            key = np.sort(np.partition(key.ravel(), key.size - case["k"])[-case["k"]:])[::-1]
            scores[b] = key
        return {"parents": None, "tokens": None, "scores": torch.from_numpy(scores)}
    if case["op"] == "reorder":
        x, parents, u = s["states"].cpu(), s["parents"].cpu().tolist(), case["used"]
        y = x.clone()
        for b, line in enumerate(parents):
            for i, j in enumerate(line):
                y[:, b, i, :, :u] = x[:, b, j, :, :u]
        return y
    lens, seen, acc, pos = host("lens"), host("seen"), host("acc"), host("pos")
    keys, values = s["keys"].cpu(), s["values"].cpu()
    out = np.zeros_like(acc)
    for b in range(case["batch"]):
        w = s["weights"][b].double().view(case["heads"], -1, case["capacity"]).cpu().numpy().sum(1)
        n, m = int(lens[b]), min(int(lens[b]), case["budget"])
        for h in range(case["heads"]):
            total = acc[b, h, :n] + w[h, :n]
            held = (pos[b, h, :n] < case["sink"]) | (pos[b, h, :n] >= seen[b] - case["recent"])
            worth = np.where(held, np.inf, total.astype(np.float32).astype(np.float64))
            kept = np.zeros(n, bool)
            kept[np.lexsort((np.arange(n), -worth))[:m]] = True
            at = np.arange(m)
            at[~kept[:m]] = m + np.flatnonzero(kept[m:])
            out[b, h, :m] = total[at]
            keys[b, h, :m], values[b, h, :m] = keys[b, h, at], values[b, h, at]
    return {"lens": None, "acc": torch.from_numpy(out), "pos": None, "keys": keys, "values": values}
