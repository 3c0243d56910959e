"""Cases of the operators that serve a batch of requests from a paged key-value cache: keys rotated and stored with their
values into the pages of each request, attention over those pages, and the log probabilities of tokens with the entropy
of their distribution and its likeliest alternatives.

`run` computes a case in its plain form (elementary torch operations), or with `own` set through the framework's entry
points: k_rope_kv_store_paged, k_attention_paged_rows and k_token_logprobs. Both take the same inputs from `prepare`.

Sizes are those of the two benchmark architectures (32/8 heads of 128 and 32/8 heads of 64, vocabulary 128256) or
generic ones."""
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HEADS = [(32, 8, 128), (32, 8, 64), (16, 16, 64), (14, 2, 64), (28, 4, 128), (8, 2, 32)]
PAGES = [8, 16, 17, 24, 32, 64, 128]


def listed():
    return [
        # ---- keys and values into their pages
        # one request's next token: the smallest step, where the launch counts
        _store("store-1x1", 32, 8, 64, 1, 1, 2048, 16, "bf16"),
        # a decode batch whose requests bring drafts, pages of a size that is no power of two
        _store("store-48x3-f16", 32, 8, 128, 48, 3, 4096, 24, "f16"),
        # the prompts of four requests, of different lengths, in one call
        _store("store-4x512", 32, 8, 128, 4, 512, 2048, 64, "bf16"),
        # ---- attention over the pages
        # one request right after a short prompt
        _attention("attention-1x1-s128", 32, 8, 64, 1, 1, 128, 16, "bf16"),
        # a small batch at a few thousand positions
        _attention("attention-8x1-s2048-f16", 32, 8, 128, 8, 1, 2048, 32, "f16"),
        # up to five rows a request (the last token and its drafts), odd lengths, pages that end inside any tile
        _attention("attention-16x5-s4099", 32, 8, 128, 16, 5, 4099, 24, "bf16"),
        # seven query heads to a key, the cache in 32 bits as the contiguous one
        _attention("attention-24x1-s3001-f32", 28, 4, 128, 24, 1, 3001, 16, "f32"),
        # a full serving batch at up to 8192 positions
        _attention("attention-64x1-s8192", 32, 8, 128, 64, 1, 8192, 64, "bf16"),
        # ---- log probabilities
        # one sampled token, a small vocabulary, no alternatives
        _logprobs("logprobs-1-v32000", 1, 32000, 0, 0),
        # a decode batch's sampled tokens, twenty alternatives each
        _logprobs("logprobs-64-v128256-top20", 64, 128256, 20, 0),
        # an odd vocabulary in longer rows, some tokens of it ruled out (-infinity)
        _logprobs("logprobs-129-v50001-top5", 129, 50001, 5, 1),
        # the tokens of a prompt
        _logprobs("logprobs-2048-v128256-top5", 2048, 128256, 5, 0),
    ]


def _store(name, heads, kv, hd, batch, rows, seq, page, dtype):
    return {"name": name, "op": "store", "heads": heads, "kv": kv, "hd": hd, "batch": batch, "rows": rows, "seq": seq,
            "page": page, "dtype": dtype}


def _attention(name, heads, kv, hd, batch, rows, seq, page, dtype):
    return {"name": name, "op": "attention", "heads": heads, "kv": kv, "hd": hd, "batch": batch, "rows": rows, "seq": seq,
            "page": page, "dtype": dtype}


def _logprobs(name, rows, vocab, top, masked):
    """masked: some tokens are ruled out, and the rows of logits are longer than the vocabulary."""
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "top": top, "masked": masked}


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["store", "attention", "logprobs"])
    while True:
        if op == "logprobs":
            c = _logprobs("", _log(rng, 1, 2048), _log(rng, 64, 200000), rng.choice([0, 1, 5, 20, 32]), rng.randint(0, 1))
        else:
            heads, kv, hd = rng.choice(HEADS)
            page, dtype, batch = rng.choice(PAGES), rng.choice(sorted(DTYPES)), _log(rng, 1, 64)
            if op == "store":
                rows = _log(rng, 1, 512)
                c = _store("", heads, kv, hd, batch, rows, rows + _log(rng, 1, 4096), page, dtype)
            else:
                rows = rng.choice([1, 1, 1, 2, 3, 5, 8])
                c = _attention("", heads, kv, hd, batch, rows, rows - 1 + _log(rng, 1, 16384), page, dtype)
        most = [work(x) for x in listed() if x["op"] == op]
        w = work(c)
        if w["bytes"] <= max(m["bytes"] for m in most) and w["flops"] <= max(m["flops"] for m in most):
            del c["name"]
            return c


def _requests(c):
    """(positions stored before, rows in use) of each request: lengths spread from a quarter of the longest to all of it,
    every number of rows; in a batch of more than three, one slot is not in use."""
    B, R, S = c["batch"], c["rows"], c["seq"]
    out = []
    for i in range(B):
        count = R if i == B - 1 else 1 + i % R
        length = S if i == B - 1 else max(count, S // 4 + (S - S // 4) * i // (B - 1))
        out.append((length - count, 0 if B > 3 and i == 1 else count))
    return out


def work(case):
    c = case
    if c["op"] == "logprobs":  # a weight of each logit (one exponential), its sum and the entropy's
        n = c["rows"] * c["vocab"]
        return {"bytes": 4 * n + 4 * c["rows"] * (3 + 2 * c["top"]), "flops": 5 * n}
    H, KV, hd, size = c["heads"], c["kv"], c["hd"], DTYPES[c["dtype"]].itemsize
    live = [(s, n) for s, n in _requests(c) if n]
    rows = sum(n for _, n in live)
    if c["op"] == "store":
        return {"bytes": rows * (4 * (2 * H + 2 * KV) * hd + 2 * KV * hd * size + 4 * 2 * hd), "flops": 3 * rows * (H + KV) * hd}
    seen = sum(s * n + n * (n + 1) // 2 for s, n in live)
    return {"bytes": 2 * KV * hd * size * sum(s + n for s, n in live) + 4 * 2 * rows * H * hd, "flops": 4 * H * hd * seen}


def _inputs(case, seed):
    c, g = case, torch.Generator("cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
    whole = lambda low, high, *shape: torch.randint(low, high, shape, device="cuda", generator=g, dtype=torch.int32)  # noqa: E731
    if c["op"] == "logprobs":
        rows, V, top = c["rows"], c["vocab"], c["top"]
        ld = V + 24 if c["masked"] else V
        logits = 3.0 * normal(rows, ld)
        if c["masked"]:
            logits = torch.where(torch.rand(logits.shape, device="cuda", generator=g) < 0.1, -math.inf, logits)
            logits[:, :1] = 0.5  # the first token is always possible
        # most of the given tokens are likely ones, as sampled ones and a prompt's are
        likely = (logits[:, :V] - torch.log(-torch.log(torch.rand(rows, V, device="cuda", generator=g).clamp(1e-7, 1 - 1e-7)))).argmax(-1)
        other = whole(0, V, rows)
        possible = logits.gather(-1, other.long()[:, None])[:, 0] > -math.inf
        tokens = torch.where((whole(0, 8, rows) == 0) & possible, other, likely.int())
        if rows > 3:
            tokens[1] = -1  # a slot of the batch that is not in use
        return {"logits": logits, "tokens": tokens, "logprobs": torch.zeros(rows, device="cuda"),
                "entropy": torch.zeros(rows, device="cuda"),
                "top_tokens": torch.zeros(rows, top, device="cuda", dtype=torch.int32),
                "top_logprobs": torch.zeros(rows, top, device="cuda")}
    B, R, H, KV, hd, page, dtype = c["batch"], c["rows"], c["heads"], c["kv"], c["hd"], c["page"], DTYPES[c["dtype"]]
    requests = torch.tensor(_requests(c), dtype=torch.int32)
    order = torch.randperm(B, generator=torch.Generator().manual_seed(seed))
    starts, counts = requests[order, 0], requests[order, 1]
    # the requests' pages lie anywhere in a pool that has some to spare; the table names none where a request has none
    width = -(-c["seq"] // page)
    used = torch.where(counts > 0, -(-(starts + counts) // page), 0)
    has = torch.arange(width) < used[:, None]
    total = int(used.sum())
    pool = total + 4
    at = torch.randperm(pool - 1, generator=torch.Generator().manual_seed(seed + 1))[:total]  # the last one is spare
    table = torch.full((B, width), -1, dtype=torch.int32)
    table[has] = at.to(torch.int32)
    s = {"table": table.cuda(), "starts": starts.cuda(), "counts": counts.cuda(), "q": 1.5 * normal(B, R, H * hd),
         "out": torch.zeros(B, R, H * hd, device="cuda")}
    for name in ("key", "value"):
        s[name] = torch.empty(pool, KV, page, hd, dtype=dtype, device="cuda")
        for p in range(0, pool, 4096):
            part = s[name][p:p + 4096]
            part.copy_(normal(*part.shape))
    if c["op"] == "store":
        s["k"], s["v"] = normal(B, R, KV * hd), normal(B, R, KV * hd)
        # a row of the table: each pair's cosine twice, then its sine with and without sign
        angle = torch.arange(c["seq"], device="cuda", dtype=torch.float64)[:, None] * \
            500000.0 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
        cos, sin = angle.cos().float(), angle.sin().float()
        s["rope"] = torch.cat([torch.stack([cos, cos], -1).flatten(1), torch.stack([-sin, sin], -1).flatten(1)], 1)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:  # what a program keeps: the cache's description and the workspace
        c, kc = case, _package()
        if c["op"] != "logprobs":
            s["cache"] = kc.paged_cache(s["key"], s["value"], s["table"])
        if c["op"] == "attention":
            s["work"] = kc.paged_attention_work(c["heads"], c["kv"], c["hd"], c["batch"], c["rows"])
    return s


def _package():
    if "llama3x_b200" not in sys.modules:
        at = Path(__file__).resolve().parents[1] / "llama3.x.c_b200"
        spec = importlib.util.spec_from_file_location("llama3x_b200", at / "__init__.py",
                                                      submodule_search_locations=[str(at)])
        module = importlib.util.module_from_spec(spec)
        sys.modules["llama3x_b200"] = module
        spec.loader.exec_module(module)
    return sys.modules["llama3x_b200"]


def run(state):
    if own:
        return _own(state)
    return {"store": _plain_store, "attention": _plain_attention, "logprobs": _plain_logprobs}[state["case"]["op"]](state)


def _own(s):
    c, kc = s["case"], _package()
    if c["op"] == "store":
        dq, dkv = c["heads"] * c["hd"], c["kv"] * c["hd"]
        kc.k_rope_kv_store_paged(s["out"], dq, s["q"], dq, s["k"], s["v"], dkv, s["cache"], s["rope"], c["seq"],
                                 s["starts"], s["counts"], c["heads"], c["kv"], c["hd"], c["batch"], c["rows"])
        return {"q": s["out"], "key": s["key"], "value": s["value"]}
    if c["op"] == "attention":
        kc.k_attention_paged_rows(s["out"], None, None, s["q"], s["cache"], s["starts"], s["counts"], s["work"],
                                  c["heads"], c["kv"], c["hd"], c["batch"], c["rows"], 0)
        return s["out"]
    top = c["top"] > 0
    kc.k_token_logprobs(s["logprobs"], s["entropy"], s["top_tokens"] if top else None, s["top_logprobs"] if top else None,
                        s["logits"], s["logits"].shape[1], s["tokens"], c["vocab"], c["rows"], c["top"])
    return {name: s[name] for name in ("logprobs", "entropy", "top_tokens", "top_logprobs")}


def _rotated(x, table, hd):
    """x [B][R][n * hd] with the table rows [B][R][2 * hd]: each pair (a, b) to (a cos - b sin, a sin + b cos)."""
    pair = x.unflatten(-1, (-1, hd // 2, 2))
    cos, sin = table[:, :, None, 0:hd:2], table[:, :, None, hd + 1::2]
    a, b = pair[..., 0], pair[..., 1]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(2)


def _plain_store(s):
    c = s["case"]
    B, R, KV, hd, page = c["batch"], c["rows"], c["kv"], c["hd"], c["page"]
    row = torch.arange(R, device="cuda")
    used = row < s["counts"][:, None]  # [B, R]
    position = torch.where(used, s["starts"][:, None] + row, 0).long()
    rope = s["rope"][position]
    q = torch.where(used[:, :, None], _rotated(s["q"], rope, hd), 0.0)
    pages = s["key"].shape[0]
    # rows out of use go to the first place of the spare page, as it is
    at = torch.where(used, s["table"].long().gather(1, position // page), pages - 1)
    slot = torch.where(used, position % page, 0)
    index = (at[:, :, None], torch.arange(KV, device="cuda"), slot[:, :, None])
    for cache, new in ((s["key"], _rotated(s["k"], rope, hd)), (s["value"], s["v"])):
        new = new.view(B, R, KV, hd).to(cache.dtype)
        cache[index] = torch.where(used[:, :, None, None], new, cache[index])
    return {"q": q, "key": s["key"], "value": s["value"]}


def _plain_attention(s):
    c = s["case"]
    B, R, H, KV, hd = c["batch"], c["rows"], c["heads"], c["kv"], c["hd"]
    G = H // KV
    where = s["table"].long().clamp(min=0)
    flat = lambda cache: cache[where].transpose(1, 2).reshape(B, KV, -1, hd).float()  # noqa: E731
    q = s["q"].view(B, R, KV, G, hd).transpose(1, 2).reshape(B, KV, R * G, hd) / math.sqrt(hd)
    scores = q @ flat(s["key"]).transpose(2, 3)  # [B, KV, R * G, S]
    row = torch.arange(R * G, device="cuda") // G
    seen = torch.arange(scores.shape[-1], device="cuda") <= (s["starts"][:, None] + row)[:, :, None]
    scores = torch.where(seen[:, None], scores, -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = (weights @ flat(s["value"])) / weights.sum(-1, keepdim=True)
    out = out.view(B, KV, R, G, hd).transpose(1, 2).reshape(B, R, H * hd)
    used = row[::G] < s["counts"][:, None]
    return torch.where(used[:, :, None], out, 0.0)  # rows out of use keep the zeros of the output buffer


def _plain_logprobs(s):
    c = s["case"]
    x = s["logits"][:, :c["vocab"]]
    used = s["tokens"] >= 0
    shifted = x - x.amax(-1, keepdim=True)
    weight = torch.exp(shifted)
    total = weight.sum(-1, dtype=torch.float64)
    log_total = torch.log(total)
    # a token that is ruled out adds nothing to the entropy
    mean = torch.where(weight > 0, weight * shifted, 0.0).sum(-1, dtype=torch.float64) / total
    at = shifted.gather(-1, s["tokens"].clamp(min=0).long()[:, None])[:, 0]
    best, places = torch.sort(shifted, dim=-1, descending=True, stable=True)  # ties: the lowest token first
    best, places = best[:, :c["top"]], places[:, :c["top"]]
    return {"logprobs": torch.where(used, at - log_total, 0.0).float(),
            "entropy": torch.where(used, log_total - mean, 0.0).float(),
            "top_tokens": torch.where(used[:, None], places, 0).int(),
            "top_logprobs": torch.where(used[:, None], best - log_total[:, None], 0.0).float()}


def exact(case, seed):
    return {"store": _exact_store, "attention": _exact_attention, "logprobs": _exact_logprobs}[case["op"]](case, _inputs(case, seed))


def _exact_store(c, s):
    KV, hd, page = c["kv"], c["hd"], c["page"]
    key, value = s["key"].double(), s["value"].double()
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    table, starts, counts = s["table"].tolist(), s["starts"].tolist(), s["counts"].tolist()
    turn = torch.view_as_complex(torch.stack([s["rope"][:, 0:hd:2], s["rope"][:, hd + 1::2]], -1).double())  # [seq, hd / 2]
    for b in range(c["batch"]):  # page by page
        first, end = starts[b], starts[b] + counts[b]
        while first < end:
            upto = min(end, (first // page + 1) * page)
            rows = slice(first - starts[b], upto - starts[b])
            angle = turn[first:upto, None]

            def turned(x):
                z = torch.view_as_complex(x.double().view(upto - first, -1, hd // 2, 2).contiguous())
                return torch.view_as_real(z * angle).reshape(upto - first, -1, hd)

            q[b, rows] = turned(s["q"][b, rows]).flatten(1)
            at, slots = table[b][first // page], slice(first % page, first % page + upto - first)
            key[at, :, slots] = turned(s["k"][b, rows]).transpose(0, 1)
            value[at, :, slots] = s["v"][b, rows].double().view(upto - first, KV, hd).transpose(0, 1)
            first = upto
    return {"q": q, "key": key, "value": value}


def _exact_attention(c, s):
    B, R, H, KV, hd, page = c["batch"], c["rows"], c["heads"], c["kv"], c["hd"], c["page"]
    out = torch.zeros(B, R, H, hd, dtype=torch.float64, device="cuda")
    q = s["q"].double().view(B, R, KV, H // KV, hd)
    table, starts, counts = s["table"].tolist(), s["starts"].tolist(), s["counts"].tolist()
    for b in range(B):  # one request at a time, its pages laid out whole
        if not counts[b]:
            continue
        n = starts[b] + counts[b]
        ids = torch.tensor(table[b][:-(-n // page)], device="cuda")
        keys, values = (x[ids].double().transpose(0, 1).flatten(1, 2)[:, :n] for x in (s["key"], s["value"]))
        scores = torch.einsum("rkgd,kpd->rkgp", q[b, :counts[b]], keys) * hd ** -0.5
        limit = starts[b] + torch.arange(counts[b], device="cuda")
        scores.masked_fill_((torch.arange(n, device="cuda") > limit[:, None])[:, None, None], -math.inf)
        out[b, :counts[b]] = torch.einsum("rkgp,kpd->rkgd", scores.softmax(-1), values).reshape(counts[b], H, hd)
    return out.view(B, R, H * hd)


def _exact_logprobs(c, s):
    rows, V, top = c["rows"], c["vocab"], c["top"]
    tokens = s["tokens"].tolist()
    out = {"logprobs": torch.zeros(rows, dtype=torch.float64, device="cuda"),
           "entropy": torch.zeros(rows, dtype=torch.float64, device="cuda"),
           "top_tokens": torch.zeros(rows, top, dtype=torch.int32, device="cuda"),
           "top_logprobs": torch.zeros(rows, top, dtype=torch.float64, device="cuda")}
    for r in range(rows):
        if tokens[r] < 0:
            continue
        row = s["logits"][r, :V]
        log_p = torch.log_softmax(row.double(), -1)
        out["logprobs"][r] = log_p[tokens[r]]
        out["entropy"][r] = torch.special.entr(log_p.exp()).sum()
        # the lowest tokens among equals: by value downwards, then by index
        edge = torch.kthvalue(-row, top).values if top else row[0]
        near = (-row <= edge).nonzero()[:, 0] if top else row[:0].long()
        picked = near[torch.argsort(-row[near], stable=True)][:top]
        out["top_tokens"][r] = picked.int()
        out["top_logprobs"][r] = log_p[picked]
    return out
