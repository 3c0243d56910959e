"""Cases of the operators that serve a batch of requests over one prompt: attention over a prefix that the batch shares,
low-rank adapters of the requests beside a shared projection, and the verification of drafted tokens.

`run` computes a case in its plain form (elementary torch operations), or with `own` set through the framework's entry
points: k_attention_shared_rows, k_lora_rows and k_verify_draft. Both take the same inputs from `prepare`.

Sizes are those of the two benchmark architectures (dim 4096, hidden 14336, 32/8 heads of 128, and dim 2048, hidden
8192, 32/8 heads of 64, vocabulary 128256) or generic ones."""
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NAMES = {"f32": "K_F32", "bf16": "K_BF16", "f16": "K_F16"}


def listed():
    return [
        # ---- attention over a shared prefix
        # two requests right after a short system prompt: the smallest step, where the launches count
        _attention("attention-2x1-p128", 32, 8, 64, 2, 1, 128, 16),
        # a small batch decoding behind a document of 2048 tokens
        _attention("attention-8x1-p2048", 32, 8, 128, 8, 1, 2048, 512),
        # five rows a request (the last token and four drafts), a prefix and a cache of odd lengths
        _attention("attention-16x5-p4099", 32, 8, 128, 16, 5, 4099, 301),
        # a full serving batch, four rows a request, behind 8192 tokens
        _attention("attention-64x4-p8192", 32, 8, 128, 64, 4, 8192, 512),
        # ---- adapters
        # one request's token through a square projection of the smaller architecture
        _lora("lora-1x2048", 1, 1, 8, 2048, 2048, "bf16", "each", 0),
        # a decode batch in which every request has its own adapter
        _lora("lora-64x4096", 64, 64, 16, 4096, 4096, "bf16", "each", 0),
        # the up projection, few adapters in no order, some rows without one, fp32 adapters of mixed ranks
        _lora("lora-33x4096x14336", 33, 5, 32, 4096, 14336, "f32", "mixed", 1),
        # the prompts of four requests in one prefill batch
        _lora("lora-2048x4096", 2048, 4, 64, 4096, 4096, "bf16", "runs", 0),
        # ---- drafts
        # one request, one draft, a small vocabulary
        _verify("verify-1x1-v32000", 1, 1, 32000, 1, 0.0),
        # one request, four drafts of a draft model
        _verify("verify-1x4-v128256", 1, 4, 128256, 1, 0.0),
        # drafts looked up in the prompt (no draft probabilities), some of the requests greedy
        _verify("verify-24x7-lookup", 24, 7, 128256, 0, 0.3),
        # a full serving batch, five drafts a request, ragged
        _verify("verify-64x5-v128256", 64, 5, 128256, 1, 0.1),
    ]


def _attention(name, heads, kv, hd, batch, rows, prefix, seq):
    return {"name": name, "op": "attention", "heads": heads, "kv": kv, "hd": hd, "batch": batch, "rows": rows,
            "prefix": prefix, "seq": seq}


def _lora(name, rows, count, rank, n, d, dtype, order, mixed):
    """order: each (row r has adapter r mod count), mixed (any adapter, one row in eight without), runs (contiguous)."""
    return {"name": name, "op": "lora", "rows": rows, "count": count, "rank": rank, "n": n, "d": d, "dtype": dtype,
            "order": order, "mixed": mixed}


def _verify(name, batch, rows, vocab, drafted, greedy):
    """drafted: 1 with the draft model's logits, 0 without; greedy: the share of requests at temperature 0."""
    return {"name": name, "op": "verify", "batch": batch, "rows": rows, "vocab": vocab, "drafted": drafted,
            "greedy": greedy}


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attention", "lora", "verify"])
    while True:
        if op == "attention":
            heads, kv, hd = rng.choice([(32, 8, 128), (32, 8, 64), (16, 16, 64), (14, 2, 64), (28, 4, 128), (8, 2, 32)])
            rows = rng.randint(1, 8)
            c = _attention("", heads, kv, hd, _log(rng, 1, 64), rows, _log(rng, 1, 16384) - 1, rows + _log(rng, 1, 1024))
        elif op == "lora":
            c = _lora("", _log(rng, 1, 2048), _log(rng, 1, 64), rng.choice([4, 8, 16, 32, 64]), 64 * _log(rng, 4, 224),
                      8 * _log(rng, 32, 1792) + rng.choice([0, 0, 0, 3]), rng.choice(sorted(DTYPES)),
                      rng.choice(["each", "mixed", "runs"]), rng.randint(0, 1))
        else:
            c = _verify("", _log(rng, 1, 64), rng.randint(0, 8), _log(rng, 512, 128256), rng.randint(0, 1),
                        rng.choice([0.0, 0.25, 1.0]))
        most = [work(x) for x in listed() if x["op"] == op]
        w = work(c)
        if w["bytes"] <= max(m["bytes"] for m in most) and w["flops"] <= max(m["flops"] for m in most):
            del c["name"]
            return c


def work(case):
    c = case
    if c["op"] == "attention":  # on average the caches are half full and so are the requests' rows
        own_rows = (c["seq"] + 1) / 2
        q = c["batch"] * (c["rows"] + 1) / 2 * c["heads"] * c["hd"]
        kv = 2 * c["kv"] * c["hd"] * (c["prefix"] + c["batch"] * own_rows)
        return {"bytes": 4 * (2 * q + kv), "flops": 4 * q * (c["prefix"] + own_rows)}
    if c["op"] == "lora":
        size = 4 if c["dtype"] == "f32" else 2
        used = min(c["count"], c["rows"])
        return {"bytes": 4 * c["rows"] * (c["n"] + 2 * c["d"]) + size * used * c["rank"] * (c["n"] + c["d"]),
                "flops": 2 * c["rows"] * c["rank"] * (c["n"] + c["d"])}
    # every row of logits that counts once (half of the drafts on average, no draft logits where a request is greedy):
    # a weight (one exponential), its sum, and for one row a request the running sum
    drafts = c["rows"] / 2
    values = c["vocab"] * c["batch"] * (drafts + 1 + (drafts * (1 - c["greedy"]) if c["drafted"] else 0))
    return {"bytes": 4 * values, "flops": 4 * values}


def _inputs(case, seed):
    c, g = case, torch.Generator("cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
    whole = lambda low, high, *shape: torch.randint(low, high, shape, device="cuda", generator=g, dtype=torch.int32)  # noqa: E731
    if c["op"] == "attention":
        B, R, S, hd = c["batch"], c["rows"], c["seq"], c["hd"]
        room = c["prefix"] + 5  # the prefix lies in a cache with room for more positions
        counts = whole(1, R + 1, B)
        counts[B // 2] = R
        if B > 3:
            counts[1] = 0  # a slot of the batch that is not in use
        return {"q": 1.5 * normal(B, R, c["heads"] * hd), "pk": normal(c["kv"], room, hd), "pv": normal(c["kv"], room, hd),
                "k": normal(B, c["kv"], S, hd), "v": normal(B, c["kv"], S, hd), "starts": whole(0, S - R + 1, B),
                "counts": counts, "out": torch.zeros(B, R, c["heads"] * hd, device="cuda")}
    if c["op"] == "lora":
        n, d, count, dtype = c["n"], c["d"], c["count"], DTYPES[c["dtype"]]
        rank = [max(1, c["rank"] >> (i % 3)) if c["mixed"] else c["rank"] for i in range(count)]
        row = torch.arange(c["rows"], device="cuda", dtype=torch.int32)
        index = {"each": row % count, "runs": row * count // c["rows"], "mixed": whole(0, count, c["rows"])}[c["order"]]
        if c["order"] == "mixed":
            index = torch.where(whole(0, 8, c["rows"]) == 0, -1, index)
        return {"x": normal(c["rows"], n), "base": normal(c["rows"], d), "out": torch.zeros(c["rows"], d, device="cuda"),
                "index": index.to(torch.int32), "a": [(normal(r, n) / math.sqrt(n)).to(dtype) for r in rank],
                "b": [(0.3 * normal(d, r)).to(dtype) for r in rank], "scale": [2.0 * 16 / (16 + i % 5) for i in range(count)]}
    B, R, V = c["batch"], c["rows"], c["vocab"]
    target = 4.0 * normal(B, R + 1, V)
    uniform = lambda *shape: torch.rand(shape, device="cuda", generator=g)  # noqa: E731
    temperature = torch.where(uniform(B) < c["greedy"], 0.0, 0.6 + 0.6 * uniform(B))
    draft = target[:, :R] + 0.8 * normal(B, R, V)
    pick = draft / temperature.clamp(min=1e-3)[:, None, None] - torch.log(-torch.log(uniform(B, R, V).clamp(1e-7, 1 - 1e-7)))
    drafted = pick.argmax(-1).to(torch.int32) if R else whole(0, V, B, 0)
    counts = whole(0, R + 1, B)
    counts[B // 2] = R
    if B > 3:
        counts[1] = -1  # a slot of the batch that is not in use
    return {"target": target, "draft": draft.contiguous() if c["drafted"] else None, "drafted": drafted, "counts": counts,
            "uniforms": uniform(B, R + 1), "temperature": temperature,
            "accepted": torch.zeros(B, device="cuda", dtype=torch.int32),
            "tokens": torch.zeros(B, R + 1, device="cuda", dtype=torch.int32)}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:  # what a program keeps: the workspaces and the adapters' table
        c, kc = case, _package()
        if c["op"] == "attention":
            s["work"] = kc.shared_attention_work(c["heads"], c["kv"], c["hd"], c["batch"], c["rows"])
        elif c["op"] == "lora":
            s["table"] = kc.lora_table(s["a"], s["b"], s["scale"])
        else:
            s["work"] = torch.empty(kc.k_verify_bytes(c["vocab"], c["batch"], c["rows"]), dtype=torch.uint8, device="cuda")
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
    return {"attention": _plain_attention, "lora": _plain_lora, "verify": _plain_verify}[state["case"]["op"]](state)


def _own(s):
    c, kc = s["case"], _package()
    if c["op"] == "attention":
        kc.k_attention_shared_rows(s["out"], None, None, s["q"], s["pk"], s["pv"], s["pk"].shape[1], c["prefix"], s["k"],
                                   s["v"], s["starts"], s["counts"], s["work"], c["heads"], c["kv"], c["hd"], c["seq"],
                                   c["batch"], c["rows"], 0)
        return s["out"]
    if c["op"] == "lora":
        kc.k_lora_rows(s["out"], c["d"], s["base"], c["d"], s["x"], c["n"], s["index"], s["table"], c["count"],
                       getattr(kc, NAMES[c["dtype"]]), c["rank"], c["n"], c["d"], c["rows"])
        return s["out"]
    kc.k_verify_draft(s["accepted"], s["tokens"], s["target"], c["vocab"], s["draft"], c["vocab"], s["drafted"],
                      s["counts"], s["uniforms"], s["temperature"], c["vocab"], c["batch"], c["rows"], s["work"])
    return {"accepted": s["accepted"], "tokens": s["tokens"]}


def _plain_attention(s):
    c = s["case"]
    B, R, H, KV, hd, P, S = c["batch"], c["rows"], c["heads"], c["kv"], c["hd"], c["prefix"], c["seq"]
    G = H // KV
    q = s["q"].view(B, R, KV, G, hd).permute(2, 0, 1, 3, 4) / math.sqrt(hd)  # [KV, B, R, G, hd]
    far = (q.reshape(KV, B * R * G, hd) @ s["pk"][:, :P].transpose(1, 2)).view(KV, B, R * G, P)
    near = (q.transpose(0, 1).reshape(B, KV, R * G, hd) @ s["k"].transpose(2, 3)).transpose(0, 1)  # [KV, B, R * G, S]
    row = torch.arange(R * G, device="cuda") // G
    seen = torch.arange(S, device="cuda") <= (s["starts"][:, None] + row)[:, :, None]  # [B, R * G, S]
    near = torch.where(seen, near, -math.inf)
    top = near.amax(-1, keepdim=True)
    if P:
        top = torch.maximum(top, far.amax(-1, keepdim=True))
    far, near = torch.exp(far - top), torch.exp(near - top)
    total = far.sum(-1, keepdim=True) + near.sum(-1, keepdim=True)
    own_v = (near.transpose(0, 1) @ s["v"]).transpose(0, 1)
    out = ((far.reshape(KV, B * R * G, P) @ s["pv"][:, :P]).view(KV, B, R * G, hd) + own_v) / total
    out = out.view(KV, B, R, G, hd).permute(1, 2, 0, 3, 4).reshape(B, R, H * hd)
    used = torch.arange(R, device="cuda") < s["counts"][:, None]
    return torch.where(used[:, :, None], out, 0.0)  # rows out of use keep the zeros of the output buffer


def _plain_lora(s):
    a, b = torch.cat(s["a"]).float(), torch.cat(s["b"], 1).float()  # every adapter's rows side by side
    ranks = torch.tensor([x.shape[0] for x in s["a"]], device="cuda")
    owner = torch.repeat_interleave(torch.arange(len(s["a"]), device="cuda"), ranks, output_size=a.shape[0])
    scale = torch.tensor(s["scale"], device="cuda")[owner]
    low = torch.where(s["index"][:, None] == owner, (s["x"] @ a.T) * scale, 0.0)
    return s["base"] + low @ b.T


def _plain_verify(s):
    c = s["case"]
    B, R, V = c["batch"], c["rows"], c["vocab"]
    greedy = s["temperature"] == 0
    warm = torch.where(greedy, 1.0, s["temperature"]).double()[:, None, None]

    def probabilities(logits):
        x = logits.double() / warm
        e = torch.exp(x - x.amax(-1, keepdim=True))
        return e / e.sum(-1, keepdim=True)

    p = probabilities(s["target"])
    place = torch.arange(V, device="cuda")
    best = torch.where(s["target"] == s["target"].amax(-1, keepdim=True), place, V).amin(-1)  # [B, R + 1]
    x = s["drafted"].long()[:, :, None]
    at_p = p[:, :R].gather(-1, x)[:, :, 0]
    if s["draft"] is not None:
        q = probabilities(s["draft"]) if R else p[:, :R]
        at_q = q.gather(-1, x)[:, :, 0]
    else:
        q, at_q = (place == x).double(), 1.0
    good = torch.where(greedy[:, None], s["drafted"] == best[:, :R], s["uniforms"][:, :R].double() * at_q < at_p)
    step = torch.arange(R, device="cuda")
    good = good & (step < s["counts"][:, None])
    accepted = torch.cumprod(good.int(), 1).sum(1)  # drafts before the first refused one
    live = s["counts"] >= 0
    rest = p.gather(1, accepted[:, None, None].expand(B, 1, V))[:, 0]
    if R:
        minus = q.gather(1, accepted.clamp(max=R - 1)[:, None, None].expand(B, 1, V))[:, 0]
        refused = accepted < s["counts"]  # the next token comes from what the draft left of the target
        rest = torch.where(refused[:, None], (rest - minus).clamp(min=0), rest)
    run_up = torch.cumsum(rest, -1)
    sampled = (run_up <= s["uniforms"][:, R].double()[:, None] * run_up[:, -1:]).sum(-1).clamp(max=V - 1)
    last = torch.where(greedy, best.gather(1, accepted[:, None])[:, 0], sampled)
    at = torch.arange(R + 1, device="cuda")
    drafted = torch.cat([s["drafted"].long(), torch.zeros(B, 1, device="cuda", dtype=torch.int64)], 1)
    tokens = torch.where(at < accepted[:, None], drafted, torch.where(at == accepted[:, None], last[:, None], -1))
    return {"accepted": torch.where(live, accepted, 0).int(), "tokens": torch.where(live[:, None], tokens, 0).int()}


def exact(case, seed):
    return {"attention": _exact_attention, "lora": _exact_lora, "verify": _exact_verify}[case["op"]](case, _inputs(case, seed))


def _exact_attention(c, s):
    B, R, H, KV, hd, P = c["batch"], c["rows"], c["heads"], c["kv"], c["hd"], c["prefix"]
    G = H // KV
    out = torch.zeros(B, R, H, hd, dtype=torch.float64, device="cuda")
    q = s["q"].double().view(B, R, H, hd)
    pk, pv = s["pk"][:, :P].double(), s["pv"][:, :P].double()
    starts, counts = s["starts"].tolist(), s["counts"].tolist()
    for b in range(B):  # one request at a time, its keys laid out whole
        if not counts[b]:
            continue
        n = starts[b] + counts[b]
        keys = torch.cat([pk, s["k"][b, :, :n].double()], 1)
        values = torch.cat([pv, s["v"][b, :, :n].double()], 1)
        at = torch.arange(P + n, device="cuda")
        qb = q[b, :counts[b]].reshape(counts[b], KV, G, hd)
        scores = torch.einsum("rkgd,kpd->rkgp", qb, keys) * hd ** -0.5
        limit = P + starts[b] + torch.arange(counts[b], device="cuda")
        scores.masked_fill_((at[None] > limit[:, None])[:, None, None], -math.inf)
        out[b, :counts[b]] = torch.einsum("rkgp,kpd->rkgd", scores.softmax(-1), values).reshape(counts[b], H, hd)
    return out.view(B, R, H * hd)


def _exact_lora(c, s):
    out = s["base"].double()
    for i, (a, b, scale) in enumerate(zip(s["a"], s["b"], s["scale"])):
        rows = (s["index"] == i).nonzero()[:, 0]
        if len(rows):
            out[rows] += scale * ((s["x"][rows].double() @ a.double().T) @ b.double().T)
    return out


def _exact_verify(c, s):
    B, R, V = c["batch"], c["rows"], c["vocab"]
    accepted = torch.zeros(B, dtype=torch.int32)
    tokens = torch.zeros(B, R + 1, dtype=torch.int32)
    counts, temperature, drafted = s["counts"].tolist(), s["temperature"].tolist(), s["drafted"].tolist()
    uniforms = s["uniforms"].tolist()
    for b in range(B):
        if counts[b] < 0:
            continue
        tokens[b] = -1
        j, last = 0, None
        while last is None:
            row = s["target"][b, j]
            if temperature[b] == 0:
                token = int((row == row.max()).nonzero()[0])
                refused = j == counts[b] or drafted[b][j] != token
                weights = None
            else:
                log_p = torch.log_softmax(row.double() / temperature[b], -1)
                refused, weights = j == counts[b], log_p.exp()
                if not refused:
                    x = drafted[b][j]
                    if s["draft"] is not None:
                        log_q = torch.log_softmax(s["draft"][b, j].double() / temperature[b], -1)
                    else:
                        log_q = torch.full_like(log_p, -math.inf)
                        log_q[x] = 0.0
                    u = uniforms[b][j]
                    refused = not (u == 0 or math.log(u) + float(log_q[x]) < float(log_p[x]))
                    if refused:
                        weights = (weights - log_q.exp()).clamp(min=0)
            if refused:
                if weights is None:
                    last = token
                else:  # the sum of what lies behind each token, from the end
                    behind = weights.flip(0).cumsum(0).flip(0) - weights
                    left = (1.0 - uniforms[b][R]) * float(weights.sum())
                    last = int((behind < left).nonzero()[0])
            else:
                tokens[b, j] = drafted[b][j]
                j += 1
        tokens[b, j] = last
        accepted[b] = j
    return {"accepted": accepted, "tokens": tokens}
