"""The serving and scoring operators: what is timed, on which inputs, and their plain forms.

Five operators around the model's key / solved-value cache and its logits:

  step      paged_decode_step: one new token per sequence over a paged cache; the token's solved
            value x_new = v - sum_t exp(s k^.k^_t - 1/s) x_t, the attention of its query heads over
            the cached tokens and itself, and the new row written into its page
  attend    paged_decode_attention: the attention of one new token over the cached tokens alone
  append    paged_append: ragged rows of new keys and solved values written into the sequences' pages
  copy      copy_pages: whole pages copied in every layer (forking a sequence, compacting the pool)
  logprobs  token_logprobs: log probabilities of given tokens, the entropy and the most likely
            alternatives of each row of logits; with "train", the gradient of the first two too

Pools are [pages, kv heads, page size, head dim] bf16 (copy: [layers, pages, ...]), block tables
[sequences, table width] int32 in a random order of the pool's pages, lengths [sequences] int32.
"""
import random

import torch

own = False


def _case(name, op, **kw):
    return {"name": name, "op": op, **kw}


def listed():
    return [
        # the first steps of one chat on the repository's decoder (32 query heads, 4 kv heads of 68): latency only
        _case("step_short", "step", batch=1, hq=32, hkv=4, dim=68, page=16, longest=37, mix=0),
        # a serving batch of that decoder: ragged contexts, some sequences just begun
        _case("step_ragged", "step", batch=24, hq=32, hkv=4, dim=68, page=64, longest=6007, mix=1),
        # the decode benchmark's batch without grouped heads over 32K cached tokens
        _case("step_32k", "step", batch=4, hq=32, hkv=32, dim=128, page=128, longest=32765, mix=0),
        # a larger ragged batch with grouped heads, empty slots among its sequences
        _case("attend_ragged", "attend", batch=48, hq=32, hkv=4, dim=128, page=32, longest=8150, mix=3),
        # one long document: 128K cached tokens, work only along the cache
        _case("attend_128k", "attend", batch=1, hq=32, hkv=4, dim=128, page=64, longest=131072, mix=0),
        # one decoded token of each of 64 sequences
        _case("append_token", "append", batch=64, hkv=4, dim=68, page=16, rows=1, longest=3000, mix=1),
        # a prefill's rows of eight prompts of different lengths, right-padded
        _case("append_prompts", "append", batch=8, hkv=4, dim=68, page=64, rows=4093, longest=500, mix=1),
        # forking: the partly filled last pages of eight sequences, in all 22 layers
        _case("copy_fork", "copy", layers=22, hkv=4, dim=68, page=64, pages=256, moved=8),
        # compacting a pool after many sequences ended
        _case("copy_compact", "copy", layers=22, hkv=4, dim=68, page=64, pages=1024, moved=400),
        # what a sampler reports of a few decoded tokens: fp32 logits, some of them banned
        _case("logprobs_sampled", "logprobs", rows=8, vocab=32000, dtype="float32", top=5, banned=0.4, train=False),
        # scoring two 4K documents with 20 alternatives a token
        _case("logprobs_score", "logprobs", rows=8190, vocab=32000, dtype="bfloat16", top=20, banned=0.0, train=False),
        # a policy's update on 4K tokens: log probabilities and entropies with the gradient of the logits
        _case("logprobs_train", "logprobs", rows=4095, vocab=32000, dtype="bfloat16", top=0, banned=0.0, train=True),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["step", "attend", "append", "copy", "logprobs", "train"])
    if op in ("step", "attend"):
        dim = rng.choice([32, 64, 68, 80, 96, 128, 128])
        hkv = rng.choice([1, 2, 4, 8, 32])
        hq = hkv * (rng.choice([1, 1, 2, 3]) if hkv == 32 else rng.choice([1, 2, 4, 7, 8, 16, 24]))
        batch = _spread(rng, 1, 96)
        # at most 1 GB of cached rows
        longest = _spread(rng, 1, min(150000, max(64, 10 ** 9 // (batch * hkv * dim * 4))))
        return {"op": op, "batch": batch, "hq": hq, "hkv": hkv, "dim": dim, "page": rng.choice([1, 16, 24, 32, 64, 128, 256]) if longest < 20000 else 64,
                "longest": longest, "mix": rng.choice([0, 1, 2, 3])}
    if op == "append":
        rows = _spread(rng, 1, 4096)
        return {"op": op, "batch": _spread(rng, 1, 64 if rows < 500 else 8), "hkv": rng.choice([1, 2, 4, 8, 32]), "dim": rng.choice([32, 64, 68, 80, 128]),
                "page": rng.choice([1, 16, 24, 64, 128]), "rows": rows, "longest": _spread(rng, 1, 2000), "mix": rng.choice([0, 1, 2])}
    if op == "copy":
        layers = rng.choice([1, 2, 7, 22])
        pages = _spread(rng, 8, 800)
        return {"op": op, "layers": layers, "hkv": rng.choice([1, 2, 4, 8]), "dim": rng.choice([32, 64, 68, 128]),
                "page": rng.choice([1, 16, 24, 64]), "pages": pages, "moved": _spread(rng, 1, pages // 2)}
    vocab = _spread(rng, 100, 200000)
    rows = _spread(rng, 1, max(2, min(9000, 130_000_000 // vocab)))
    return {"op": "logprobs", "rows": rows, "vocab": vocab, "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"]),
            "top": 0 if op == "train" else rng.choice([0, 1, 5, 20, 50]), "banned": rng.choice([0.0, 0.0, 0.3, 0.9]) if vocab > 1000 else 0.0, "train": op == "train"}


def _lengths(case):
    """Cached tokens of each sequence: the case's own, whatever the seed. mix 0: all the longest; 1: uneven; 2: uneven, one long among short ones; 3: uneven, some none."""
    rng, n, longest = random.Random(case["mix"] * 1000 + case["batch"]), case["batch"], case["longest"]
    if case["mix"] == 0:
        return [longest] * n
    if case["mix"] == 2:
        return [longest] + [_spread(rng, 1, max(1, longest // 16)) for _ in range(n - 1)]
    got = [longest] + [_spread(rng, 1, longest) if rng.random() < 0.3 else rng.randint(1, longest) for _ in range(n - 1)]
    return [0 if case["mix"] == 3 and i % 7 == 3 else v for i, v in enumerate(got)]


def _counts(case):
    """New rows of each sequence (append)."""
    rng = random.Random(case["batch"] + case["rows"])
    return [case["rows"] if i == 0 or case["mix"] == 0 else rng.randint(0 if case["mix"] == 2 else 1, case["rows"]) for i in range(case["batch"])]


def _tables(case, room, seed):
    """A block table that gives every sequence the pages for `room` of its tokens, scattered over a pool with some pages to spare."""
    page = case["page"]
    need = [-(-r // page) for r in room]
    total = sum(need) + 3
    order = list(range(total))
    random.Random(seed).shuffle(order)
    table, at = torch.full((len(need), max(1, max(need)) + 1), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table.cuda(), total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *shape: torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16)
    s = {"case": case}
    if case["op"] in ("step", "attend", "append"):
        d, h = case["dim"], case["hkv"]
        lens = _lengths(case)
        new = _counts(case) if case["op"] == "append" else [1] * case["batch"]
        s["block_table"], pages = _tables(case, [a + n for a, n in zip(lens, new)], seed)
        s["lengths"] = torch.tensor(lens, dtype=torch.int32).cuda()
        # keys that lean the same way within a head, as trained ones do, so that the solve's sum is not lost next to v
        lean = rn(1, h, 1, d)
        s["key_pages"] = rn(pages, h, case["page"], d).mul_(0.8).add_(lean, alpha=0.6)
        s["x_pages"] = rn(pages, h, case["page"], d)
        if case["op"] == "append":
            # the projections' layout: [batch, rows, heads, dim] seen as [batch, heads, rows, dim]
            s["key"] = rn(case["batch"], case["rows"], h, d).transpose(1, 2)
            s["x"] = rn(case["batch"], h, case["rows"], d)
            s["counts"] = torch.tensor(new, dtype=torch.int32).cuda()
        else:
            s["scale"] = d ** -0.5
            s["query"] = rn(case["batch"], 1, case["hq"], d).transpose(1, 2)
            s["key"] = (rn(case["batch"], h, 1, d) * 0.8 + 0.6 * lean).transpose(1, 2).contiguous().transpose(1, 2)
            s["value"] = rn(case["batch"], 1, h, d).transpose(1, 2)
        return s
    if case["op"] == "copy":
        shape = (case["layers"], case["pages"], case["hkv"], case["page"], case["dim"])
        s["key_pages"], s["x_pages"] = rn(*shape), rn(*shape)
        order = list(range(case["pages"]))
        random.Random(seed).shuffle(order)
        s["src"], s["dst"] = order[:case["moved"]], order[case["moved"]:2 * case["moved"]]
        return s
    dtype = getattr(torch, case["dtype"])
    # a peaked distribution over a noisy floor, as a trained model's rows are
    logits = torch.randn(case["rows"], case["vocab"], generator=g, device="cuda", dtype=dtype).mul_(2.0)
    hot = torch.randint(case["vocab"], (case["rows"], 1), generator=g, device="cuda")
    hot = (hot + torch.arange(24, device="cuda") * (case["vocab"] // 24)) % case["vocab"]
    logits.scatter_add_(1, hot, torch.rand(case["rows"], 24, generator=g, device="cuda").mul_(9.0).to(dtype))
    tokens = hot[:, 0].clone()
    if case["banned"]:
        ban = torch.rand(case["rows"], case["vocab"], generator=g, device="cuda") < case["banned"]
        logits.masked_fill_(ban.scatter_(1, hot, False), float("-inf"))
    if case["rows"] > 2:
        tokens[case["rows"] // 2] = -100
    s["logits"], s["tokens"], s["top"] = logits, tokens, case["top"]
    if case["train"]:
        s["logits"].requires_grad_(True)
        s["grad_logprobs"] = torch.randn(case["rows"], generator=g, device="cuda")
        s["grad_entropy"] = torch.randn(case["rows"], generator=g, device="cuda").mul_(0.1)
    return s


def _rows(pool, table):
    """The tokens of every sequence side by side: [sequences, heads, table width x page size, dim] in 32 bits."""
    got = pool[table.clamp(min=0).long()].permute(0, 2, 1, 3, 4)
    return got.reshape(got.shape[0], got.shape[1], -1, got.shape[-1]).float()


def _attention(z, x):
    """softmax over the last axis of z (-inf: not seen) times x; rows that see nothing are zero."""
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, torch.matmul(p, x) / torch.where(total > 0, total, torch.ones_like(total)), torch.zeros((), device=z.device))


def _plain_decode(s):
    case = s["case"]
    b, hq, hkv, d = case["batch"], case["hq"], case["hkv"], case["dim"]
    k, x = _rows(s["key_pages"], s["block_table"]), _rows(s["x_pages"], s["block_table"])
    seen = torch.arange(k.shape[2], device=k.device) < s["lengths"][:, None]
    seen = seen[:, None, None, :]
    k, x = k * seen.transpose(2, 3), x * seen.transpose(2, 3)
    q = s["query"].float().reshape(b, hkv, hq // hkv, d)
    z = (torch.matmul(q, k.transpose(2, 3)) * s["scale"]).masked_fill(~seen, float("-inf"))
    if case["op"] == "attend":
        return _attention(z, x).reshape(b, 1, hq, d).to(torch.bfloat16)
    kn, vn = s["key"].float(), s["value"].float()
    unit = lambda t: t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-5)
    e = torch.exp(torch.matmul(unit(kn), unit(k).transpose(2, 3)) * s["scale"] - 1.0 / s["scale"]) * seen
    x_new = (vn - torch.matmul(e, x)).to(torch.bfloat16)
    z_new = torch.matmul(q, kn.transpose(2, 3)) * s["scale"]
    o = _attention(torch.cat([z, z_new], -1), torch.cat([x, x_new.float()], 2)).reshape(b, 1, hq, d).to(torch.bfloat16)
    at = s["lengths"].long()
    page = s["block_table"].gather(1, (at // case["page"])[:, None]).long()[:, 0]
    s["key_pages"][page, :, at % case["page"]] = s["key"][:, :, 0]
    s["x_pages"][page, :, at % case["page"]] = x_new[:, :, 0]
    return {"o": o, "x_new": x_new, "key_pages": s["key_pages"], "x_pages": s["x_pages"]}


def _plain_append(s):
    case = s["case"]
    n = torch.arange(case["rows"], device="cuda")
    at = s["lengths"].long()[:, None] + n
    new = n < s["counts"][:, None]
    page = s["block_table"].gather(1, (at // case["page"]).clamp(max=s["block_table"].shape[1] - 1)).long()
    b, r = new.nonzero(as_tuple=True)
    page, at = page[b, r], at[b, r] % case["page"]
    s["key_pages"][page, :, at] = s["key"][b, :, r]
    s["x_pages"][page, :, at] = s["x"][b, :, r]
    return {"key_pages": s["key_pages"], "x_pages": s["x_pages"]}


def _plain_copy(s):
    src, dst = torch.tensor(s["src"]).cuda(), torch.tensor(s["dst"]).cuda()
    s["key_pages"][:, dst] = s["key_pages"][:, src]
    s["x_pages"][:, dst] = s["x_pages"][:, src]
    return {"key_pages": s["key_pages"], "x_pages": s["x_pages"]}


def _plain_logprobs(s):
    logits, tokens = s["logits"].detach().float(), s["tokens"]
    given = tokens >= 0
    at = tokens.clamp(min=0)[:, None]
    shifted = logits - logits.amax(-1, keepdim=True)
    e = torch.exp(shifted)
    total = e.sum(-1, keepdim=True)
    logp = shifted - torch.log(total)
    p = e / total
    plogp = torch.where(p > 0, p * logp, torch.zeros((), device=p.device))
    entropy = -plogp.sum(-1)
    chosen = torch.where(given, logp.gather(1, at)[:, 0], torch.zeros((), device=p.device))
    out = {"logprobs": chosen, "entropy": entropy}
    if s["top"]:
        bits = (logits + 0.0).view(torch.int32)
        order = bits ^ ((bits >> 31) & 0x7FFFFFFF)
        keys = (order.long() << 32) + (0xFFFFFFFF - torch.arange(logits.shape[1], device=logits.device))
        out["top_tokens"] = 0xFFFFFFFF - (torch.topk(keys, s["top"], sorted=True).values & 0xFFFFFFFF)
        out["top_logprobs"] = logp.gather(1, out["top_tokens"])
    if s["case"]["train"]:
        g = torch.where(given, s["grad_logprobs"], torch.zeros((), device=p.device))[:, None]
        d = -p * g - s["grad_entropy"][:, None] * (plogp + p * entropy[:, None])
        out["grad"] = d.scatter_add_(1, at, g).to(s["logits"].dtype)
    return out


def run(s):
    case = s["case"]
    if not own:
        return {"step": _plain_decode, "attend": _plain_decode, "append": _plain_append, "copy": _plain_copy, "logprobs": _plain_logprobs}[case["op"]](s)
    import lucid_b200 as lb
    if case["op"] == "step":
        o, x_new = lb.paged_decode_step(s["query"], s["key"], s["value"], s["key_pages"], s["x_pages"], s["block_table"], s["lengths"], s["scale"], 1e-5)
        return {"o": o, "x_new": x_new, "key_pages": s["key_pages"], "x_pages": s["x_pages"]}
    if case["op"] == "attend":
        return lb.paged_decode_attention(s["query"], s["key_pages"], s["x_pages"], s["block_table"], s["lengths"], s["scale"])
    if case["op"] == "append":
        lb.paged_append(s["key"], s["x"], s["key_pages"], s["x_pages"], s["block_table"], s["lengths"], s["counts"])
        return {"key_pages": s["key_pages"], "x_pages": s["x_pages"]}
    if case["op"] == "copy":
        lb.copy_pages(s["key_pages"], s["x_pages"], s["src"], s["dst"])
        return {"key_pages": s["key_pages"], "x_pages": s["x_pages"]}
    got = lb.token_logprobs(s["logits"], s["tokens"], top=s["top"])
    out = {"logprobs": got.logprobs, "entropy": got.entropy}
    if s["top"]:
        out["top_tokens"], out["top_logprobs"] = got.top_tokens, got.top_logprobs
    if case["train"]:
        out["grad"], = torch.autograd.grad([got.logprobs, got.entropy], [s["logits"]], [s["grad_logprobs"], s["grad_entropy"]])
        out["logprobs"], out["entropy"] = got.logprobs.detach(), got.entropy.detach()
    return out


def work(case):
    if case["op"] in ("step", "attend"):
        b, hq, h, d, step = case["batch"], case["hq"], case["hkv"], case["dim"], case["op"] == "step"
        cached = sum(_lengths(case))
        ends = b * (2 * hq + (5 * h if step else 0)) * d * 2  # query, output; new key, value, solved value, the two rows written
        return {"bytes": cached * h * d * 4 + cached // case["page"] * 4 + ends, "flops": 4 * cached * d * (hq + (h if step else 0)) + (2 * cached * d * h if step else 0)}
    if case["op"] == "append":
        return {"bytes": 2 * sum(_counts(case)) * case["hkv"] * case["dim"] * 4, "flops": 0}
    if case["op"] == "copy":
        return {"bytes": 2 * case["moved"] * case["layers"] * case["hkv"] * case["page"] * case["dim"] * 4, "flops": 0}
    size = 4 if case["dtype"] == "float32" else 2
    n = case["rows"] * case["vocab"]
    return {"bytes": n * size * (2 if case["train"] else 1) + case["rows"] * (16 + 12 * case["top"] + (8 if case["train"] else 0)), "flops": n * (10 if case["train"] else 5)}


def exact(case, seed):
    if case["op"] in ("append", "copy"):
        return None
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        z = s["logits"].detach().double()
        lse = torch.logsumexp(z, -1, keepdim=True)
        logp = z - lse
        given = s["tokens"] != -100
        q = logp.exp()
        h = torch.nan_to_num(q * logp, nan=0.0).sum(-1).neg()
        chosen = logp.take_along_dim(s["tokens"].clamp(min=0)[:, None], 1)[:, 0].where(given, 0.0)
        out = {"logprobs": chosen, "entropy": h}
        if case["top"]:
            rank = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
            out["top_tokens"], out["top_logprobs"] = None, logp.take_along_dim(rank, 1)
        if case["train"]:
            hot = torch.zeros_like(q)
            hot[torch.arange(case["rows"], device="cuda"), s["tokens"].clamp(min=0)] = 1.0
            up = s["grad_logprobs"].double() * given
            out["grad"] = up[:, None] * (hot - q) - s["grad_entropy"].double()[:, None] * q * (torch.nan_to_num(logp, neginf=0.0) + h[:, None])
        return out
    group, page = case["hq"] // case["hkv"], case["page"]
    outs, solved = [], []
    for b, n in enumerate(_lengths(case)):
        where = torch.arange(n, device="cuda")
        ids = s["block_table"][b].long()[where // page] if n else where
        k = s["key_pages"][ids, :, where % page].double().transpose(0, 1)
        x = s["x_pages"][ids, :, where % page].double().transpose(0, 1)
        q = s["query"][b, :, 0].double().reshape(case["hkv"], group, -1)
        if case["op"] == "step":
            kn, vn = s["key"][b].double(), s["value"][b].double()
            cos = (kn @ k.mT) / (kn.square().mean(-1, keepdim=True) + 1e-5).sqrt() / (k.square().mean(-1)[:, None] + 1e-5).sqrt()
            xn = vn - (cos * s["scale"] - 1.0 / s["scale"]).exp() @ x
            solved.append(xn)
            k, x = torch.cat([k, kn], 1), torch.cat([x, xn.to(torch.bfloat16).double()], 1)
        outs.append((torch.softmax(q @ k.mT * s["scale"], -1) @ x).reshape(1, case["hq"], -1))
    if case["op"] == "attend":
        return torch.stack(outs)
    return {"o": torch.stack(outs), "x_new": torch.stack(solved), "key_pages": None, "x_pages": None}
