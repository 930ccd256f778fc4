"""Operators for serving many requests in one batch, as cases to measure: cross-attention to encoder states of another
length (shared, ragged, with regions) and low-rank adapters of many requests beside one shared projection.

`run` computes a case in its plain form (elementary torch operations in fp32, one rounding at the end) or, with `own` set,
through stable_diffusion_amd.engine.  `exact` is the definition in fp64, request by request."""
import math

import torch

own = False

DEV = "cuda"
H16 = torch.float16


# ------------------------------------------------------------------------------------------------------------ the cases
def listed():
    att = dict(op="attention", kv_heads=0, dim=64, regions=0)
    lor = dict(op="lora", groups=1, bias=False, residual=False, mixed=False)
    return [
        # the widest level of the UNet at 768 x 768, one prompt of 77 tokens for each of two images
        dict(att, name="attn 96x96 to 77", batch=2, contexts=2, heads=5, nq=9216, nkv=77),
        # sixteen samples of four prompts that chain up to three windows of 77 tokens, on the 24 x 24 level
        dict(att, name="attn 24x24 shared 231", batch=16, contexts=4, heads=20, nq=576, nkv=231),
        # regional prompts: each key and each latent position belongs to some of 4 regions, some positions to none
        dict(att, name="attn 48x48 regions 154", batch=4, contexts=4, heads=10, nq=2304, nkv=154, regions=4),
        # the 48 x 48 level reading the states of a whole 96 x 96 reference picture
        dict(att, name="attn 48x48 to 9216", batch=2, contexts=2, heads=10, nq=2304, nkv=9216),
        # one new token for each of eight requests over long encoder states, four query heads on each key head
        dict(att, name="attn 1 to 4096", batch=8, contexts=8, heads=16, kv_heads=4, dim=128, nq=1, nkv=4096),
        # a head width that no tile divides, odd lengths
        dict(att, name="attn 80 wide 1001 to 333", batch=4, contexts=3, heads=8, dim=80, nq=1001, nkv=333),
        # to_q of the widest level, an adapter for each of two images
        dict(lor, name="lora 96x96 to_q", requests=2, rows=9216, k=320, n=320, rank=16, adapters=2),
        # the fused q|k|v projection of the 48 x 48 level, eight images with their adapters: three low-rank pairs side by side
        dict(lor, name="lora 48x48 qkv", requests=8, rows=2304, k=640, n=1920, groups=3, rank=8, adapters=8),
        # to_out of the 24 x 24 level with its bias and the residual stream
        dict(lor, name="lora 24x24 to_out", requests=4, rows=576, k=1280, n=1280, rank=64, adapters=4, bias=True, residual=True),
        # a single token of a single request: latency
        dict(lor, name="lora 1 token", requests=1, rows=1, k=1024, n=1024, rank=16, adapters=4, bias=True),
        # the next token of each of 64 requests, every one with an adapter of its own
        dict(lor, name="lora 64 tokens", requests=64, rows=1, k=1024, n=4096, rank=32, adapters=64, bias=True),
        # the tokens of fifteen prompts packed row by row in no order, some with no adapter
        dict(lor, name="lora 1155 mixed rows", requests=1155, rows=1, k=1024, n=1024, rank=128, adapters=5, bias=True, mixed=True),
    ]


# no drawn case costs more than the largest listed one: its operations (attention to 9216 keys), its bytes in the plain form
MOST_SCORES = 2 * 10 * 2304 * 9216
MOST_PRODUCT = 8 * 2304 * 640 * 1920


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        while True:
            kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 10, 20])
            share = rng.choice([1, 1, 1, 2, 4, 8])
            batch = _log(rng, 1, 16)
            c = dict(op="attention", batch=batch, contexts=rng.choice([1, batch, rng.randint(1, batch)]), heads=kv_heads * share, kv_heads=kv_heads,
                     dim=rng.choice([32, 40, 64, 64, 64, 80, 96, 128, 160, 256]), nq=_log(rng, 1, 9216), nkv=_log(rng, 1, 9216),
                     regions=rng.choice([0, 0, 1, 3, 32]))
            if c["heads"] <= 32 and c["batch"] * c["heads"] * c["nq"] * c["nkv"] * c["dim"] <= MOST_SCORES * 64 and \
                    c["batch"] * c["heads"] * (c["nq"] + c["nkv"]) * c["dim"] <= 1 << 27:
                return c
    while True:
        mixed = rng.random() < 0.4
        requests, rows = (_log(rng, 1, 2048), 1) if mixed else (_log(rng, 1, 16), _log(rng, 1, 9216))
        groups = rng.choice([1, 1, 2, 3])
        c = dict(op="lora", requests=requests, rows=rows, k=8 * _log(rng, 8, 640), n=8 * groups * _log(rng, 8, 640 // groups), groups=groups,
                 rank=rng.choice([8, 8, 16, 16, 24, 32, 64, 128]), adapters=_log(rng, 1, 64), bias=rng.random() < 0.5, residual=rng.random() < 0.5, mixed=mixed)
        if requests * rows * c["k"] * c["n"] <= MOST_PRODUCT and c["adapters"] * c["rank"] <= 2048 and requests * rows <= 18432:
            return c


# ------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(DEV)
    g.manual_seed(int(seed))
    normal = lambda *shape, std=1.0: (torch.randn(shape, generator=g, device=DEV) * std).to(H16)
    ints = lambda lo, hi, *shape: torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    c = dict(case)
    if c["op"] == "attention":
        b, n, h, d = c["batch"], c["contexts"], c["heads"], c["dim"]
        kvh = c["kv_heads"] or h
        # keys and values leave one projection side by side; every context has states of its own length, the first the longest
        lens = ints(1, c["nkv"] + 1, n)
        lens[0] = c["nkv"]
        s = dict(case=c, q=normal(b, c["nq"], h * d, std=1.5), kv=normal(n, c["nkv"], 2 * kvh * d), lens=lens,
                 index=(torch.arange(b, device=DEV, dtype=torch.int32) if n == b else ints(0, n, b)), query_regions=None, key_regions=None)
        if c["regions"]:
            # about one position in eight lies in no region, some tokens in none either; the others in one region or two
            def sets(*shape):
                one = torch.bitwise_left_shift(torch.ones(shape, dtype=torch.int64, device=DEV), ints(0, c["regions"], *shape).long())
                two = torch.bitwise_left_shift(torch.ones(shape, dtype=torch.int64, device=DEV), ints(0, c["regions"], *shape).long())
                v = one | torch.where(ints(0, 2, *shape) == 1, two, torch.zeros_like(two))
                v = torch.where(ints(0, 8, *shape) == 0, torch.zeros_like(v), v)
                return torch.where(v >= 1 << 31, v - (1 << 32), v).to(torch.int32)
            s["query_regions"], s["key_regions"] = sets(b, c["nq"]), sets(n, c["nkv"])
        return s
    m, k, n, r, na, gr = c["requests"] * c["rows"], c["k"], c["n"], c["rank"], c["adapters"], c["groups"]
    if c["mixed"]:
        ids = ints(-1, na, c["requests"])               # -1: no adapter
    else:
        ids = (torch.randperm(max(na, c["requests"]), generator=g, device=DEV)[:c["requests"]] % na).to(torch.int32)
    return dict(case=c, x=normal(m, k), w=normal(n, k, std=k ** -0.5), a=normal(na, gr * r, k, std=k ** -0.5), b=normal(na, n, r, std=r ** -0.5),
                scale=torch.rand((na,), generator=g, device=DEV) + 0.25, ids=ids,
                bias=torch.randn((n,), generator=g, device=DEV) if c["bias"] else None, residual=normal(m, n) if c["residual"] else None)


# ------------------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _own_attention(state) if state["case"]["op"] == "attention" else _own_lora(state)
    return _plain_attention(state) if state["case"]["op"] == "attention" else _plain_lora(state)


def _plain_attention(s):
    c, index = s["case"], s["index"].long()
    b, h, d, nq, nkv = c["batch"], c["heads"], c["dim"], c["nq"], c["nkv"]
    kvh = c["kv_heads"] or h
    q = s["q"].float().view(b, nq, kvh, h // kvh, d).permute(0, 2, 3, 1, 4).reshape(b, kvh, -1, d)
    k, v = s["kv"].float().view(-1, nkv, 2, kvh, d)[index].permute(2, 0, 3, 1, 4)
    seen = (torch.arange(nkv, device=q.device)[None] < s["lens"][index][:, None]).view(b, 1, 1, 1, nkv)
    if s["query_regions"] is not None:
        seen = seen & ((s["query_regions"].view(b, 1, 1, nq, 1) & s["key_regions"][index].view(b, 1, 1, 1, nkv)) != 0)
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(d ** -0.5).view(b, kvh, h // kvh, nq, nkv)
    scores.masked_fill_(~seen, -math.inf)
    p = scores.sub_(scores.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, kvh, -1, nkv), v).view(b, kvh, h // kvh, nq, d) / total.masked_fill(total == 0, 1.0)   # nothing seen: zeros
    return o.permute(0, 3, 1, 2, 4).reshape(b, nq, h * d).to(H16)


def _plain_lora(s):
    c, x, ids = s["case"], s["x"].float(), s["ids"]
    n, r, na, gr = c["n"], c["rank"], c["adapters"], c["groups"]
    y = torch.matmul(x, s["w"].float().t())
    # every row through every adapter, all but its own one times zero: two products instead of a loop over adapters
    mine = (ids.repeat_interleave(c["rows"])[:, None] == torch.arange(na, device=ids.device)[None]) * s["scale"]
    t = torch.matmul(x, s["a"].float().view(-1, c["k"]).t()).view(-1, na, gr, r) * mine[:, :, None, None]
    up = s["b"].float().view(na, gr, n // gr, r).permute(1, 0, 3, 2).reshape(gr, na * r, n // gr)
    y += torch.bmm(t.permute(2, 0, 1, 3).reshape(gr, -1, na * r), up).permute(1, 0, 2).reshape(-1, n)
    if s["bias"] is not None:
        y += s["bias"]
    if s["residual"] is not None:
        y += s["residual"].float()
    return y.to(H16)


def _own_attention(s):
    from stable_diffusion_amd import engine as E
    c = s["case"]
    b, h, d, nq, nkv = c["batch"], c["heads"], c["dim"], c["nq"], c["nkv"]
    kvh = c["kv_heads"] or h
    kv = E.Act(s["kv"], c["contexts"], 1, nkv, 2 * kvh * d)
    o = E.cross_attention(E.Act(s["q"], b, 1, nq, h * d), kv.cols(0, kvh * d), kv.cols(kvh * d, kvh * d), h, kv_heads=kvh, dim=d, index=s["index"],
                          lens=s["lens"], query_regions=s["query_regions"], key_regions=s["key_regions"])
    return o.buf


def _own_lora(s):
    from stable_diffusion_amd import engine as E
    c, m = s["case"], s["x"].shape[0]
    res = None if s["residual"] is None else E.Act(s["residual"].view(1, m, -1), 1, 1, m, c["n"])
    y = E.lora_gemm(E.Act(s["x"].view(1, m, -1), 1, 1, m, c["k"]), s["w"], c["n"], E.LoraPack(s["a"], s["b"], s["scale"]), s["ids"], bias=s["bias"], residual=res)
    return y.buf.view(m, c["n"])


# ------------------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    c = case
    if c["op"] == "attention":
        kvh = c["kv_heads"] or c["heads"]
        # lengths are uniform, the first context's is the full one: (the mean of) the keys that are read and attended to
        used = min(c["contexts"], c["batch"])
        keys = (c["nkv"] + (c["contexts"] - 1) * (c["nkv"] + 1) / 2) / c["contexts"]
        moved = 2 * 2 * c["batch"] * c["nq"] * c["heads"] * c["dim"] + 2 * 2 * used * keys * kvh * c["dim"]
        if c["regions"]:
            moved += 4 * c["batch"] * c["nq"] + 4 * used * keys
        return {"bytes": moved, "flops": 4 * c["batch"] * c["heads"] * c["nq"] * keys * c["dim"]}
    m, used = c["requests"] * c["rows"], min(c["adapters"], c["requests"])
    rank = c["rank"]
    moved = 2 * (m * c["k"] + c["n"] * c["k"] + m * c["n"] * (2 if c["residual"] else 1) + used * rank * (c["groups"] * c["k"] + c["n"])) + 4 * c["requests"]
    return {"bytes": moved + (4 * c["n"] if c["bias"] else 0), "flops": 2 * m * (c["n"] * c["k"] + c["groups"] * rank * c["k"] + rank * c["n"])}


# ------------------------------------------------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "attention":
        h, d, kvh = c["heads"], c["dim"], c["kv_heads"] or c["heads"]
        out = torch.zeros((c["batch"], c["nq"], h * d), dtype=torch.float64, device=DEV)
        for i, (ctx, lens) in enumerate(zip(s["index"].tolist(), s["lens"][s["index"].long()].tolist())):
            hidden = None
            if s["query_regions"] is not None:
                hidden = torch.bitwise_and(s["query_regions"][i].view(-1, 1), s["key_regions"][ctx, :lens].view(1, -1)) == 0
            for head in range(h):
                at = head * kvh // h * d
                logit = s["q"][i, :, head * d:(head + 1) * d].double() @ s["kv"][ctx, :lens, at:at + d].double().t() / math.sqrt(d)
                if hidden is not None:
                    logit[hidden] = -math.inf
                weight = torch.nan_to_num(torch.softmax(logit, dim=1), nan=0.0)           # a row of -inf alone: no weight at all
                out[i, :, head * d:(head + 1) * d] = weight @ s["kv"][ctx, :lens, kvh * d + at:kvh * d + at + d].double()
        return out
    x, per = s["x"].double(), c["n"] // c["groups"]
    out = x @ s["w"].double().t()
    owner = s["ids"].long()[torch.arange(x.shape[0], device=DEV) // c["rows"]]
    for j in range(c["adapters"]):
        rows = torch.nonzero(owner == j).flatten()
        if not rows.numel():
            continue
        low = float(s["scale"][j]) * (x[rows] @ s["a"][j].double().t())
        for g in range(c["groups"]):
            out[rows, g * per:(g + 1) * per] += low[:, g * c["rank"]:(g + 1) * c["rank"]] @ s["b"][j, g * per:(g + 1) * per].double().t()
    if s["bias"] is not None:
        out = out + s["bias"].double()
    if s["residual"] is not None:
        out = out + s["residual"].double()
    return out
