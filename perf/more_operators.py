"""Cases of the serving cache and of token scores: what generating from and scoring with the language model need.

``append``  new tokens' routed keys and dense values into the pages of a cache
``attend``  outer routed attention of a chunk of new tokens (one, a few, or a long chunk) over a paged cache
``score``   log probabilities of given tokens with the entropy and the top alternatives, and their backward pass

``run`` computes a case in elementary torch operations in 32 bits, or, where ``own`` is true, through
``double_attention_b200``.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def _paged(op: str, sequences: int, new: int, context: int, branches: int, maps: int, routing: int, dim: int, page: int,
           dtype: str, ragged: bool) -> dict:
    return {"op": op, "sequences": sequences, "new": new, "context": context, "branches": branches, "maps": maps,
            "routing": routing, "dim": dim, "page": page, "dtype": dtype, "ragged": ragged}


def listed() -> list[dict]:
    return [
        # a decoding step of 64 sequences: each one's new key and value
        {"name": "append decode", **_paged("append", 64, 1, 500, 1, 1, 256, 512, 64, "bf16", True)},
        # prefill of 16 prompts of up to 1024 tokens with four branches
        {"name": "append prefill", **_paged("append", 16, 1024, 0, 4, 4, 128, 512, 64, "bf16", True)},
        # one token of one short conversation
        {"name": "attend token", **_paged("attend", 1, 1, 511, 1, 1, 256, 512, 16, "bf16", False)},
        # a decoding step of 64 conversations of up to 8192 tokens
        {"name": "attend decode", **_paged("attend", 64, 1, 8191, 1, 1, 256, 512, 64, "bf16", True)},
        # one token behind a very long document, wide routing
        {"name": "attend long", **_paged("attend", 1, 1, 131071, 1, 1, 512, 512, 128, "bf16", False)},
        # five drafted tokens of eight sequences checked at once, two maps
        {"name": "attend drafts", **_paged("attend", 8, 5, 2003, 2, 2, 256, 512, 32, "fp16", True)},
        # a prompt taken in chunks: 512 more tokens of a long document
        {"name": "attend chunk", **_paged("attend", 1, 512, 32768, 1, 1, 256, 512, 64, "bf16", False)},
        # a batch of uneven chunks over uneven caches, four maps
        {"name": "attend uneven chunks", **_paged("attend", 6, 700, 4001, 4, 4, 128, 512, 64, "fp16", True)},
        # the alternatives to one decoded token, small vocabulary
        {"name": "score token", "op": "score", "rows": 1, "vocabulary": 2048, "dtype": "fp32", "top": 5,
         "masked": False, "backward": False},
        # a decoding step of 64 sequences, wide uneven vocabulary with entries that a grammar rules out
        {"name": "score decode", "op": "score", "rows": 64, "vocabulary": 50021, "dtype": "bf16", "top": 20,
         "masked": True, "backward": False},
        # scoring 16 prompts of 1024 tokens
        {"name": "score prompts", "op": "score", "rows": 16384, "vocabulary": 2048, "dtype": "bf16", "top": 8,
         "masked": False, "backward": False},
        # a policy's training step over 64 sequences of 1024 tokens: log probabilities and entropy, with their gradient
        {"name": "score training", "op": "score", "rows": 65536, "vocabulary": 2048, "dtype": "bf16", "top": 0,
         "masked": False, "backward": True},
    ]


def _log(rng, lo: int, hi: int) -> int:
    n = min(max(int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))), lo), hi)
    return n


def draw(rng) -> dict:
    op = rng.choice(["append", "attend", "attend", "attend", "score", "score"])
    if op == "score":
        vocabulary = _log(rng, 64, 100000)
        backward = rng.random() < 0.5
        return {"op": op, "rows": min(_log(rng, 1, 65536), 67_000_000 // vocabulary), "vocabulary": vocabulary,
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "top": 0 if backward else rng.choice([0, 1, 5, 8, 20, 32]),
                "masked": rng.random() < 0.3, "backward": backward}
    branches, maps, routing = rng.choice([(1, 1, 64), (1, 1, 128), (1, 1, 256), (1, 1, 256), (1, 1, 512), (2, 1, 256),
                                          (1, 2, 256), (2, 2, 256), (2, 2, 128), (4, 4, 128), (4, 4, 128), (4, 2, 64)])
    dim, page = rng.choice([128, 256, 512, 512]), rng.choice([16, 32, 64, 128])
    dtype, ragged = rng.choice(["bf16", "fp16"]), rng.random() < 0.5
    if op == "append":
        sequences, new = _log(rng, 1, 64), _log(rng, 1, 1024)
        return _paged(op, sequences, min(new, max(1, 16384 // sequences)), rng.randrange(0, 500), branches, maps, routing,
                      dim, page, dtype, ragged)
    new = 1 if rng.random() < 0.3 else _log(rng, 1, 2048)
    context = 0 if rng.random() < 0.1 else _log(rng, 1, 131072)
    sequences = max(1, min(_log(rng, 1, 64), 300_000 // (context + new), 16_000_000 // (new * (context + new))))
    new = max(1, min(new, 16_000_000 // (context + new)))
    return _paged(op, sequences, new, context, branches, maps, routing, dim, page, dtype, ragged)


# ----------------------------------------------------------------------------- inputs
def _sizes(case: dict) -> tuple[list[int], list[int]]:
    """Tokens in the cache before the call, and new tokens, of each sequence."""
    held, new = [], []
    for b in range(case["sequences"]):
        spread = b * 2654435761 % 1000 / 1000 if case["ragged"] else 0.0
        held.append(int(case["context"] * (1 - 0.5 * spread)))
        new.append(max(1, int(case["new"] * (1 - 0.7 * spread))))
    return held, new


def _unit(g: torch.Generator, rows: int, width: int, centres: torch.Tensor) -> torch.Tensor:
    """Routed vectors: of unit length, several kinds of them."""
    kind = torch.randint(0, centres.shape[0], (rows,), generator=g, device="cuda")
    x = centres[kind] + torch.randn(rows, width, generator=g, device="cuda")
    return x / x.norm(dim=1, keepdim=True)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    s: dict = {"case": case}
    if case["op"] == "score":
        rows, width = case["rows"], case["vocabulary"]
        logits = 2.5 * torch.randn(rows, width, generator=g, device="cuda")
        s["tokens"] = torch.randint(0, width, (rows,), generator=g, device="cuda")
        # (a trained model gives its own tokens a good share)
        logits.scatter_add_(1, s["tokens"][:, None], torch.full((rows, 1), 6.0, device="cuda"))
        if case["masked"]:
            ruled_out = torch.rand(width, generator=g, device="cuda") < 0.3
            ruled_out = ruled_out[None].expand(rows, width).scatter(1, s["tokens"][:, None], False)
            logits.masked_fill_(ruled_out, -math.inf)
        s["logits"] = logits.to(DTYPES[case["dtype"]])
        if case["backward"]:
            s["d_log_probs"] = torch.randn(rows, generator=g, device="cuda")
            s["d_entropy"] = torch.full((rows,), -0.01, device="cuda")
            s["logits"].requires_grad_()
        return s
    dtype = DTYPES[case["dtype"]]
    branches, routing, page = case["branches"], case["routing"], case["page"]
    held, new = _sizes(case)
    total, sequences = sum(new), case["sequences"]
    need = [-(-(h + n) // page) for h, n in zip(held, new)]
    pages = sum(need) + 3  # the cache has room left
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    s["table"] = torch.zeros(sequences, max(need), dtype=torch.int32, device="cuda")
    taken = 0
    for b, n in enumerate(need):
        s["table"][b, :n] = order[taken:taken + n]
        taken += n
    s["lengths"] = torch.tensor(held, dtype=torch.int32, device="cuda")
    s["starts"] = torch.tensor([sum(new[:b]) for b in range(sequences + 1)], dtype=torch.int32, device="cuda")
    s["max_new"] = max(new)
    centres = 0.8 * torch.randn(12, routing, generator=g, device="cuda")
    s["key_pages"] = _unit(g, pages * page * branches, routing, centres).to(dtype).view(pages, page, branches, routing)
    s["value_pages"] = torch.randn(pages, page, case["dim"], generator=g, device="cuda").to(dtype)
    s["routed"] = _unit(g, 2 * branches * total, routing, centres).to(dtype).view(2, branches, 1, total, routing)
    s["values"] = torch.randn(total, case["dim"], generator=g, device="cuda").to(dtype)
    if case["op"] == "attend":
        s["scales"] = 16.0 * torch.exp(0.05 * torch.randn(case["maps"], generator=g, device="cuda"))
        s["weights"] = None
        if case["maps"] > 1:
            s["weights"] = torch.softmax(0.3 * torch.randn(case["maps"], generator=g, device="cuda"), dim=0)
    return s


# ----------------------------------------------------------------------------- plain form
def _places(s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """Each packed new token's sequence, and its position there."""
    starts = s["starts"].long()
    token = torch.arange(s["values"].shape[0], device="cuda")
    sequence = torch.searchsorted(starts[1:], token, right=True)
    return sequence, s["lengths"].long()[sequence] + token - starts[sequence]


def _plain_append(s: dict):
    page = s["case"]["page"]
    sequence, position = _places(s)
    row = s["table"].long()[sequence, position // page] * page + position % page
    s["key_pages"].flatten(0, 1)[row] = s["routed"][1, :, 0].transpose(0, 1)
    s["value_pages"].flatten(0, 1)[row] = s["values"]
    return {"key_pages": s["key_pages"], "value_pages": s["value_pages"]}


def _plain_attend(s: dict):
    case = s["case"]
    maps, branches, routing = case["maps"], case["branches"], case["routing"]
    page, starts, lengths = case["page"], s["starts"].long(), s["lengths"].long()
    sequence, position = _places(s)
    # every sequence's cache side by side, [sequences, length, ...]
    where = (s["table"].long()[:, :, None] * page + torch.arange(page, device="cuda")).flatten(1)
    keys = s["key_pages"].flatten(0, 1)[where].float()
    values = s["value_pages"].flatten(0, 1)[where].float()
    there = torch.arange(where.shape[1], device="cuda") < (lengths + starts[1:] - starts[:-1])[:, None]
    values = torch.where(there[..., None], values, torch.zeros_like(values))
    # the new tokens padded to [sequences, most new tokens, ...]
    slot = torch.arange(s["max_new"], device="cuda")
    token = (starts[:-1, None] + slot).clamp(max=sequence.shape[0] - 1)
    query = s["routed"][0, :, 0][:, token].float()  # [branches, sequences, most new, routing]
    sees = torch.arange(where.shape[1], device="cuda") <= (lengths[:, None] + slot)[..., None]
    if branches >= maps:  # a map's score adds up its branches
        group = branches // maps
        q = query.view(maps, group, *query.shape[1:]).permute(2, 0, 3, 1, 4).flatten(3)
        k = keys.view(*keys.shape[:2], maps, group * routing).permute(0, 2, 3, 1)
    else:
        group, repeat = 1, maps // branches
        q = query.permute(1, 0, 2, 3).repeat_interleave(repeat, dim=1)
        k = keys.permute(0, 2, 3, 1).repeat_interleave(repeat, dim=1)
    score = (q @ k) * (s["scales"] / math.sqrt(group))[:, None, None]
    score = score.masked_fill(~sees[:, None], -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True))
    weight = weight / weight.sum(-1, keepdim=True)
    if s["weights"] is not None:
        weight = weight * s["weights"][:, None, None]
    out = weight.sum(1) @ values  # [sequences, most new, dim]
    return {"y": out[sequence, position - lengths[sequence]].to(DTYPES[case["dtype"]])}


def _plain_score(s: dict):
    case, tokens = s["case"], s["tokens"][:, None]
    x = s["logits"].detach().float()
    x = x - x.amax(1, keepdim=True)
    e = torch.exp(x)
    log_total = torch.log(e.sum(1, keepdim=True))
    lp = x - log_total
    p = torch.exp(lp)
    finite = torch.where(p > 0, lp, torch.zeros_like(lp))
    entropy = -(p * finite).sum(1)
    out = {"log_probs": lp.gather(1, tokens)[:, 0], "entropy": entropy}
    if case["top"]:
        order = torch.sort(s["logits"].detach(), dim=1, descending=True, stable=True).indices[:, :case["top"]]
        out |= {"top_log_probs": lp.gather(1, order), "top_tokens": order}
    if case["backward"]:
        d = -p * (s["d_log_probs"][:, None] + s["d_entropy"][:, None] * (finite + entropy[:, None]))
        d.scatter_add_(1, tokens, s["d_log_probs"][:, None])
        out["d_logits"] = d.to(s["logits"].dtype)
    return out


# ----------------------------------------------------------------------------- the framework's operators
def _framework(s: dict):
    import double_attention_b200 as da

    case = s["case"]
    if case["op"] == "score":
        made = da.token_log_probs(s["logits"], s["tokens"], top=case["top"])
        out = {"log_probs": made.log_probs, "entropy": made.entropy}
        if case["top"]:
            out |= {"top_log_probs": made.top_log_probs, "top_tokens": made.top_tokens}
        if case["backward"]:
            out["d_logits"], = torch.autograd.grad((made.log_probs, made.entropy), s["logits"],
                                                   (s["d_log_probs"], s["d_entropy"]))
            out = {name: t.detach() for name, t in out.items()}
        return out
    batch = da.PagedBatch(s["table"], s["lengths"], s["starts"], s["max_new"])
    if case["op"] == "append":
        da.append_paged(s["routed"][1, :, 0], s["values"], s["key_pages"], s["value_pages"], batch)
        return {"key_pages": s["key_pages"], "value_pages": s["value_pages"]}
    return {"y": da.routed_attention_paged(s["routed"][0, :, 0], s["key_pages"], s["value_pages"], batch, s["scales"],
                                           s["weights"])}


def run(state: dict):
    if own:
        return _framework(state)
    return {"append": _plain_append, "attend": _plain_attend, "score": _plain_score}[state["case"]["op"]](state)


# ----------------------------------------------------------------------------- work and definition
def work(case: dict) -> dict:
    if case["op"] == "score":
        n, size = case["rows"] * case["vocabulary"], BYTES[case["dtype"]]
        return {"bytes": n * size * (2 if case["backward"] else 1) + case["rows"] * (16 + 12 * case["top"]),
                "flops": n * (14 if case["backward"] else 7)}
    held, new = _sizes(case)
    wide = case["branches"] * case["routing"]
    token = 2 * (wide + case["dim"])
    if case["op"] == "append":
        return {"bytes": 2 * sum(new) * token, "flops": sum(new)}
    pairs = sum(n * h + n * (n + 1) // 2 for h, n in zip(held, new))
    scored = max(wide, case["maps"] * case["routing"])  # a repeated branch is scored again, with another scale
    return {"bytes": sum(h + n for h, n in zip(held, new)) * token + sum(new) * token,
            "flops": pairs * (2 * (min(scored, wide) + case["dim"]) + 4 * case["maps"])}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "score":
        if case["rows"] * case["vocabulary"] > 200_000_000:
            return None
        x = s["logits"].detach().to(f64)
        lse = torch.logsumexp(x, 1)
        rows = torch.arange(case["rows"], device="cuda")
        p = torch.softmax(x, 1)
        entropy = torch.special.entr(p).sum(1)
        out = {"log_probs": x[rows, s["tokens"]] - lse, "entropy": entropy}
        if case["top"]:
            # the largest first, and of equal ones the one that comes first
            best = [sorted(range(len(r)), key=lambda i, r=r: (-r[i], i))[:case["top"]] for r in x.tolist()] \
                if x.numel() <= 4_000_000 else None
            if best is None:
                ranked = torch.argsort(x, dim=1, descending=True, stable=True)[:, :case["top"]]
            else:
                ranked = torch.tensor(best, device="cuda")
            out |= {"top_log_probs": x.gather(1, ranked) - lse[:, None], "top_tokens": ranked}
        if case["backward"]:
            # H = -sum p log p falls by p_i (log p_i + H) with logit i, and log p_t rises by [i = t] - p_i
            d = -s["d_entropy"].to(f64)[:, None] * (entropy[:, None] * p - torch.special.entr(p))
            d -= s["d_log_probs"].to(f64)[:, None] * p
            d[rows, s["tokens"]] += s["d_log_probs"].to(f64)
            out["d_logits"] = d
        return out
    held, new = _sizes(case)
    page, maps, branches = case["page"], case["maps"], case["branches"]
    keys, values = s["key_pages"], s["value_pages"]
    table, first = s["table"].tolist(), 0
    made = []
    if case["op"] == "append":
        keys, values = keys.to(f64), values.to(f64)
        for b in range(case["sequences"]):
            slots = torch.tensor([table[b][t // page] * page + t % page for t in range(held[b], held[b] + new[b])],
                                 device="cuda")
            for h in range(branches):
                keys.view(-1, branches, case["routing"])[slots, h] = s["routed"][1, h, 0, first:first + new[b]].to(f64)
            values.view(-1, case["dim"])[slots] = s["values"][first:first + new[b]].to(f64)
            first += new[b]
        return {"key_pages": keys, "value_pages": values}
    for b in range(case["sequences"]):
        length = held[b] + new[b]
        used = torch.tensor(table[b][:-(-length // page)], device="cuda")
        k = keys[used].reshape(-1, branches, case["routing"])[:length].to(f64)
        v = values[used].reshape(-1, case["dim"])[:length].to(f64)
        later = torch.ones(new[b], length, dtype=torch.bool, device="cuda").triu(held[b] + 1)
        y = torch.zeros(new[b], case["dim"], dtype=f64, device="cuda")
        for m in range(maps):
            mine = range(m * branches // maps, max((m + 1) * branches // maps, m * branches // maps + 1))
            logit = sum(s["routed"][0, h, 0, first:first + new[b]].to(f64) @ k[:, h].t() for h in mine)
            logit = (logit * s["scales"][m].to(f64) / math.sqrt(len(mine))).masked_fill(later, -math.inf)
            y += torch.softmax(logit, 1) @ v * (1.0 if s["weights"] is None else s["weights"][m].to(f64))
        made.append(y)
        first += new[b]
    return {"y": torch.cat(made)}
