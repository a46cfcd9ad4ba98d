"""Measured cases of the 16-bit expert products and of the low-rank adapters.

Three operators of ``glmserve_b200.ops``:

  grouped_gemm        y[p] = x[rows[p]] W[e]^T for the rows p of expert e's segment (ragged segments)
  moe_expert_ffn_w16  sum_k w[t,k] * down(silu(gate x) * up x) over 16-bit expert weights
  lora_add            y[t] += scale[a] * B[a] (A[a] x[t]) with the adapter a of every row

``run`` computes them in plain 32-bit torch operations, or with ``own`` set calls the library.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


# ---- cases --------------------------------------------------------------------------------

def listed():
    return [
        # one decoded token, eight experts of the 1024-wide layer: latency
        dict(name="grouped 1 token", op="grouped", rows=8, tokens=1, experts=32, k=1024, n=512, skew=0.0, type="bf16"),
        # a decode batch on the 32 experts that one of eight GPUs holds of the 6144-wide layer, gate projection
        dict(name="grouped decode", op="grouped", rows=64, tokens=64, experts=32, k=6144, n=2048, skew=0.0, type="bf16"),
        # a ragged batch: sizes off every tile, skewed loads, experts without a row
        dict(name="grouped ragged", op="grouped", rows=1777, tokens=777, experts=13, k=1032, n=1515, skew=1.1, type="fp16"),
        # a prompt chunk of 8192 tokens, top-2 of eight experts of the 4096-wide layer, down projection
        dict(name="grouped prefill", op="grouped", rows=16384, tokens=8192, experts=8, k=2048, n=4096, skew=0.5, type="bf16"),
        # one decoded token through the whole expert FFN: latency
        dict(name="ffn 1 token", op="ffn", tokens=1, topk=8, experts=32, of=32, hidden=1024, inter=512, skew=0.0, type="bf16"),
        # a decode batch on one of eight expert-parallel shards: most slots belong to other GPUs (id -1)
        dict(name="ffn decode shard", op="ffn", tokens=64, topk=8, experts=32, of=256, hidden=6144, inter=2048, skew=0.0, type="bf16"),
        # small odd layer
        dict(name="ffn odd", op="ffn", tokens=333, topk=3, experts=5, of=5, hidden=520, inter=264, skew=1.1, type="fp16"),
        # a prompt chunk of 8192 tokens through the 4096-wide layer, top-2 of eight experts
        dict(name="ffn prefill", op="ffn", tokens=8192, topk=2, experts=8, of=8, hidden=4096, inter=2048, skew=0.3, type="bf16"),
        # one token of one request
        dict(name="lora 1 token", op="lora", tokens=1, adapters=8, k=1024, n=1024, rank=16, bare=0.0, type="bf16", out="f32"),
        # a decode batch of 64 requests with an adapter each, beside a 6144-wide projection
        dict(name="lora decode", op="lora", tokens=64, adapters=64, k=6144, n=6144, rank=16, bare=0.1, type="bf16", out="f32"),
        # a ragged batch with ranks that differ, rows without an adapter, 16-bit output
        dict(name="lora ragged", op="lora", tokens=517, adapters=21, k=1032, n=2050, rank=24, bare=0.3, type="fp16", out="fp16"),
        # prompt chunks of a few requests in one batch
        dict(name="lora prefill", op="lora", tokens=8192, adapters=8, k=6144, n=6144, rank=64, bare=0.1, type="bf16", out="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["grouped", "ffn", "lora"])
    dtype = rng.choice(["bf16", "fp16"])
    if kind == "grouped":
        k, n = 8 * _log(rng, 32, 512), _log(rng, 128, 4096)
        tokens = _log(rng, 1, 8192)
        rows = max(1, min(16384, int(tokens * rng.uniform(1, 8))))
        return dict(op="grouped", rows=rows, tokens=tokens, experts=rng.randint(1, 32), k=k, n=n,
                    skew=rng.choice([0.0, 0.5, 1.1]), type=dtype)
    if kind == "ffn":
        experts = rng.randint(2, 32)
        topk = rng.randint(1, min(8, experts))
        tokens = _log(rng, 1, 16384 // topk)
        # a shard has slots of its own unless the batch is tiny
        of = experts * (rng.choice([1, 1, 4]) if tokens >= 32 else 1)
        return dict(op="ffn", tokens=tokens, topk=topk, experts=experts, of=of, hidden=8 * _log(rng, 32, 512),
                    inter=8 * _log(rng, 16, 256), skew=rng.choice([0.0, 0.3, 1.1]), type=dtype)
    return dict(op="lora", tokens=_log(rng, 1, 8192), adapters=rng.randint(1, 64), k=8 * _log(rng, 32, 768),
                n=_log(rng, 256, 6144), rank=_log(rng, 4, 64), bare=rng.choice([0.0, 0.1, 0.5]), type=dtype,
                out=rng.choice(["f32", dtype]))


# ---- inputs -------------------------------------------------------------------------------

def _counts(rows, groups, skew):
    """Rows of each group: Zipf-like shares, the same for every seed (the seed only says which group is which)."""
    share = (np.arange(groups) + 1.0) ** -skew
    return np.random.default_rng(rows * 1009 + groups).multinomial(rows, share / share.sum())


def _normal(gen, shape, scale, dtype):
    t = torch.empty(shape, dtype=dtype, device=DEVICE)
    t.normal_(0.0, scale, generator=gen)
    return t


def _segments(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    order = np.random.default_rng(seed)
    dtype = TYPES[case["type"]]
    if case["op"] == "grouped":
        counts = order.permutation(_counts(case["rows"], case["experts"], case["skew"]))
        return dict(op="grouped", x=_normal(gen, (case["tokens"], case["k"]), 1.0, dtype),
                    w=_normal(gen, (case["experts"], case["n"], case["k"]), 0.02, dtype),
                    offsets=_segments(counts), cap=int(counts.max()),
                    rows=torch.randint(case["tokens"], (case["rows"],), generator=gen, device=DEVICE, dtype=torch.int32))
    if case["op"] == "ffn":
        n, of, h, i, e = (case[k] for k in ("tokens", "of", "hidden", "inter", "experts"))
        # tokens choose distinct experts by noisy scores; experts of other GPUs are id -1 here
        lean = torch.tensor(order.permutation(-case["skew"] * np.log(np.arange(of) + 1.0)), device=DEVICE)
        noise = torch.rand((n, of), generator=gen, device=DEVICE, dtype=torch.float64).clamp_(1e-12, 1 - 1e-12)
        ids = (lean - (-noise.log()).log()).topk(case["topk"], dim=1).indices.to(torch.int32)
        ids = torch.where(ids < e, ids, -1).contiguous()
        weight = torch.rand((n, case["topk"]), generator=gen, device=DEVICE) + 0.1
        weight = (2.5 * weight / weight.sum(1, keepdim=True)).contiguous()
        cap = int(torch.bincount(ids.flatten().long() + 1, minlength=e + 1)[1:].max())
        return dict(op="ffn", x=_normal(gen, (n, h), 1.0, dtype), ids=ids, weight=weight, cap=max(1, cap),
                    gate=_normal(gen, (e, i, h), 0.02, dtype), up=_normal(gen, (e, i, h), 0.02, dtype),
                    down=_normal(gen, (e, h, i), 0.02, dtype))
    n, count, r = case["tokens"], case["adapters"], case["rank"]
    # requests in any order; a share of the rows has no adapter
    which = torch.from_numpy(order.integers(0, count, n))
    which[torch.from_numpy(order.random(n)) < case["bare"]] = count
    rows = torch.argsort(which, stable=True)[: int((which < count).sum())]
    counts = torch.bincount(which, minlength=count + 1)[:count].numpy()
    ranks = torch.from_numpy(order.integers(max(1, r // 2), r + 1, count)).to(torch.int32)
    return dict(op="lora", y=_normal(gen, (n, case["n"]), 1.0, TYPES[case["out"]]), x=_normal(gen, (n, case["k"]), 1.0, dtype),
                a=_normal(gen, (count, r, case["k"]), 0.02, dtype), b=_normal(gen, (count, case["n"], r), 0.02, dtype),
                offsets=_segments(counts), rows=rows.to(torch.int32).to(DEVICE), cap=max(1, int(counts.max())),
                ranks=ranks.to(DEVICE), scales=(16.0 / ranks.float()).to(DEVICE))


# ---- the plain form -----------------------------------------------------------------------

def _by_group(x, offsets, cap, count):
    """Rows p < count of x, laid out [group, place, :] with zeros behind a group's last row; and each row's place."""
    p = torch.arange(count, device=x.device)
    group = torch.bucketize(p, offsets[1:].long(), right=True)
    place = p - offsets.long()[group]
    padded = x.new_zeros((offsets.numel() - 1, cap, x.shape[1]))
    padded[group, place] = x[:count]
    return padded, group, place


def _plain_grouped(s):
    x, group, place = _by_group(s["x"].float()[s["rows"].long()], s["offsets"], s["cap"], s["rows"].numel())
    return torch.bmm(x, s["w"].float().transpose(1, 2))[group, place].to(s["x"].dtype)


def _plain_ffn(s):
    n, topk = s["ids"].shape
    e = s["gate"].shape[0]
    slot = torch.where(s["ids"] < 0, e, s["ids"]).flatten().long()    # group e: slots of other GPUs
    order = torch.argsort(slot, stable=True)
    offsets = torch.searchsorted(slot[order], torch.arange(e + 1, device=slot.device))
    group = slot[order]
    place = torch.arange(n * topk, device=slot.device) - offsets[group]
    kept = (group < e)[:, None]
    group, place = group.clamp(max=e - 1), place.clamp(max=s["cap"] - 1)
    x = torch.where(kept, s["x"].float()[order // topk], 0.0)
    padded = x.new_zeros((e, s["cap"], x.shape[1])).index_put_((group, place), x, accumulate=True)
    g = torch.bmm(padded, s["gate"].float().transpose(1, 2))
    h = g / (1.0 + torch.exp(-g)) * torch.bmm(padded, s["up"].float().transpose(1, 2))
    y = torch.where(kept, torch.bmm(h, s["down"].float().transpose(1, 2))[group, place], 0.0)
    rows = torch.empty_like(y)
    rows[order] = y
    return (rows.view(n, topk, -1) * s["weight"][..., None]).sum(1).to(s["x"].dtype)


def _plain_lora(s):
    rows = s["rows"].long()
    if not rows.numel():
        return s["y"]
    used = (torch.arange(s["a"].shape[1], device=rows.device) < s["ranks"][:, None])[:, :, None]
    x, group, place = _by_group(s["x"].float()[rows], s["offsets"], s["cap"], rows.numel())
    v = torch.bmm(x, torch.where(used, s["a"].float(), 0.0).transpose(1, 2)) * s["scales"][:, None, None]
    d = torch.bmm(v, torch.where(used.transpose(1, 2), s["b"].float(), 0.0).transpose(1, 2))[group, place]
    s["y"][rows] = (s["y"][rows].float() + d).to(s["y"].dtype)
    return s["y"]


def run(state):
    if own:
        from glmserve_b200 import ops
        if state["op"] == "grouped":
            return ops.grouped_gemm(state["x"], state["w"], state["offsets"], rows=state["rows"])
        if state["op"] == "ffn":
            return ops.moe_expert_ffn_w16(state["x"], state["ids"], state["weight"], state["gate"], state["up"], state["down"])
        return ops.lora_add(state["y"], state["x"], state["a"], state["b"], state["offsets"], state["rows"],
                            ranks=state["ranks"], scales=state["scales"])
    return {"grouped": _plain_grouped, "ffn": _plain_ffn, "lora": _plain_lora}[state["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------

def work(case):
    if case["op"] == "grouped":
        rows, k, n = case["rows"], case["k"], case["n"]
        hit = int((_counts(rows, case["experts"], case["skew"]) > 0).sum())
        return {"bytes": 2 * (min(rows, case["tokens"]) * k + hit * n * k + rows * n) + 4 * (rows + case["experts"] + 1),
                "flops": 2 * rows * k * n}
    if case["op"] == "ffn":
        n, topk, e, of, h, i = (case[k] for k in ("tokens", "topk", "experts", "of", "hidden", "inter"))
        share = (np.arange(of) + 1.0) ** -case["skew"]
        missed = np.clip(1.0 - topk * share / share.sum(), 0.0, 1.0) ** n
        hit = min(float(e), e - e / of * missed.sum())
        rows = n * topk * e / of
        return {"bytes": 2 * (2 * n * h + hit * 3 * h * i) + 8 * n * topk, "flops": 6 * rows * h * i}
    n, k, out = case["tokens"], case["k"], case["n"]
    rows = n * (1.0 - case["bare"])
    rank = 0.75 * case["rank"]                      # ranks are spread over [rank / 2, rank]
    hit = case["adapters"] * (1.0 - (1.0 - 1.0 / case["adapters"]) ** rows)
    size = 4 if case["out"] == "f32" else 2
    return {"bytes": rows * (2 * k + 2 * size * out) + hit * rank * 2 * (k + out), "flops": 2 * rows * rank * (k + out)}


# ---- the definition in 64 bits --------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lora":
        y, at = s["y"].double(), s["offsets"].tolist()
        for a, r in enumerate(s["ranks"].tolist()):
            t = s["rows"][at[a]:at[a + 1]].long()
            y[t] += float(s["scales"][a]) * ((s["x"][t].double() @ s["a"][a, :r].double().T) @ s["b"][a, :, :r].double().T)
        return y
    if case["op"] == "grouped":
        at = s["offsets"].tolist()
        y = torch.zeros((case["rows"], case["n"]), dtype=torch.float64, device=DEVICE)
        for e in range(case["experts"]):
            y[at[e]:at[e + 1]] = s["x"][s["rows"][at[e]:at[e + 1]].long()].double() @ s["w"][e].double().T
        return y
    out = torch.zeros((case["tokens"], case["hidden"]), dtype=torch.float64, device=DEVICE)
    for e in range(case["experts"]):
        t, k = (s["ids"] == e).nonzero(as_tuple=True)
        x = s["x"][t].double()
        h = torch.nn.functional.silu(x @ s["gate"][e].double().T) * (x @ s["up"][e].double().T)
        out.index_add_(0, t, s["weight"][t, k].double()[:, None] * (h @ s["down"][e].double().T))
    return out
