"""Benchmark cases of the serving operators beside the persistent kernel: K/V rows into a paged
cache (with the position rotation on the way), attention of one new token over that cache, and
log probabilities of given tokens with entropy and top alternatives.

Every case runs in two forms.  With `own` false `run` computes the operator from elementary
torch operations in 32 bits, rounded once at the end; with `own` true it makes the calls a user
of yirage_b200 makes.  `exact` restates each operator in 64 bits.

Head counts, head sizes, vocabularies, page sizes and contexts are those of the model shapes and
benchmarks in this repository (32/8, 32/4 and 64/8 heads of 128, a tensor-parallel shard of 8/1,
vocabularies of 128256 and 151936, pages of 64, 256 and 4096 tokens), with smaller, odd and
ragged ones around them.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one request's new token on its way into the cache: the smallest call of a decode step
        dict(name="append_step_1", op="append", dtype="bf16", table="bf16", requests=1, ctx=512,
             new=1, ragged=False, hq=32, hkv=8, dim=128, rot=128, page=64, packed=True, norm=False, lens=1),
        # a full decode batch, tables in 32 bits, 64 query heads
        dict(name="append_step_64", op="append", dtype="fp16", table="fp32", requests=64, ctx=2048,
             new=1, ragged=False, hq=64, hkv=8, dim=128, rot=128, page=64, packed=True, norm=False, lens=2),
        # prompts of several requests, cut at odd places, with the q/k norm in front of the rotation
        dict(name="append_prompts_norm", op="append", dtype="bf16", table="bf16", requests=7, ctx=900,
             new=611, ragged=True, hq=32, hkv=4, dim=128, rot=128, page=64, packed=False, norm=True, lens=3),
        # long prompts handed over by another engine in one call
        dict(name="append_prompts_32k", op="append", dtype="bf16", table="bf16", requests=16, ctx=0,
             new=2048, ragged=False, hq=32, hkv=8, dim=128, rot=128, page=256, packed=True, norm=False, lens=4),
        # one short conversation: latency
        dict(name="decode_1x513", op="decode", dtype="bf16", requests=1, ctx=513, ragged=False, hq=32,
             hkv=8, dim=128, page=64, window=0, lens=5),
        # the attention benchmark of this repository: 8 requests at 4096 tokens
        dict(name="decode_8x4096", op="decode", dtype="bf16", requests=8, ctx=4096, ragged=False, hq=32,
             hkv=8, dim=128, page=64, window=0, lens=6),
        # a serving batch of very different lengths, one slot of it empty, in small pages
        dict(name="decode_64_ragged", op="decode", dtype="fp16", requests=64, ctx=8192, ragged=True, hq=64,
             hkv=8, dim=128, page=16, window=0, lens=7),
        # one very long context on a rank that holds a single K/V head
        dict(name="decode_1x131072_mqa", op="decode", dtype="bf16", requests=1, ctx=131072, ragged=False,
             hq=8, hkv=1, dim=128, page=4096, window=0, lens=8),
        # the answer's token of one request with its five best alternatives
        dict(name="logprobs_1x128256", op="logprobs", dtype="bf16", rows=1, vocab=128256, pad=768, top=5,
             masked=False),
        # a decode batch, twenty alternatives each
        dict(name="logprobs_64x151936", op="logprobs", dtype="bf16", rows=64, vocab=151936, pad=1664, top=20,
             masked=False),
        # logits in 32 bits of an odd width, part of the vocabulary ruled out in every row
        dict(name="logprobs_333x50021", op="logprobs", dtype="fp32", rows=333, vocab=50021, pad=0, top=8,
             masked=True),
        # scoring a long prompt: the log probability of every token, no alternatives
        dict(name="logprobs_4096x128256", op="logprobs", dtype="bf16", rows=4096, vocab=128256, pad=768, top=0,
             masked=False),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "decode", "logprobs"))
    hq, hkv = rng.choice(((32, 8), (64, 8), (32, 4), (8, 1), (16, 16), (8, 2), (20, 4), (48, 8)))
    dim = rng.choice((64, 128, 128, 128, 256))
    page = rng.choice((16, 48, 64, 64, 256, 4096))
    lens = rng.randrange(1 << 30)
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if op == "append":
        requests = _log_uniform(rng, 1, 256)
        new = 1 if rng.random() < 0.4 else _log_uniform(rng, 1, max(1, 16384 // requests))
        return dict(op=op, dtype=dtype, table=rng.choice((dtype, "fp32")), requests=requests,
                    ctx=_log_uniform(rng, 1, 4000), new=new, ragged=rng.random() < 0.5, hq=hq, hkv=hkv,
                    dim=dim, rot=rng.choice((dim, dim, dim // 2)), page=page, packed=rng.random() < 0.5,
                    norm=rng.random() < 0.3, lens=lens)
    if op == "decode":
        requests = _log_uniform(rng, 1, 128)
        # tokens x heads x dim stays below what the ragged batch of listed() has at most
        most = max(2, min(131072, 64 * 8192 * 8 * 128 // (2 * requests * hkv * dim)))
        return dict(op=op, dtype=dtype, requests=requests, ctx=_log_uniform(rng, 1, most),
                    ragged=rng.random() < 0.6, hq=hq, hkv=hkv, dim=dim, page=page,
                    window=rng.choice((0, 0, 0, _log_uniform(rng, 1, 4096))), lens=lens)
    rows = _log_uniform(rng, 1, 2048)
    vocab = _log_uniform(rng, 1000, min(160000, 2048 * 128256 // rows))
    return dict(op=op, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), rows=rows, vocab=vocab,
                pad=rng.choice((0, 0, 1, rng.randrange(2, 2048))), top=rng.choice((0, 1, 5, 8, 20, 32)),
                masked=rng.random() < 0.3)


# ------------------------------------------------------------------------------------ inputs
def _plan(case):
    """(length before the call, new tokens) of every request, on the host."""
    r = random.Random(case["lens"])
    n = case["requests"]
    ctx = [r.randint(0, case["ctx"]) if case["ragged"] else case["ctx"] for _ in range(n)]
    if case["op"] == "decode":
        if case["ragged"] and n > 1:
            ctx[r.randrange(n)] = 0          # a slot without a request
        return ctx, [0] * n
    new = [r.randint(1, 2 * case["new"] - 1) if case["ragged"] and case["new"] > 1 else case["new"]
           for _ in range(n)]
    return ctx, new


def _tables(case, g, dev):
    """Page tables of the batch, pages of all requests in one random order over the pool."""
    ctx, new = _plan(case)
    page = case["page"]
    total = [c + n for c, n in zip(ctx, new)]
    pages = [(t + page - 1) // page for t in total]
    pool = sum(pages) + 1
    indptr, qo = [0], [0]
    for p, n in zip(pages, new):
        indptr.append(indptr[-1] + p)
        qo.append(qo[-1] + n)
    last = [(t - 1) % page + 1 if t else 0 for t in total]
    i32 = dict(dtype=torch.int32, device=dev)
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    meta = {"qo_indptr_buffer": torch.tensor(qo, **i32),
            "paged_kv_indptr_buffer": torch.tensor(indptr, **i32),
            "paged_kv_indices_buffer": order,
            "paged_kv_last_page_len_buffer": torch.tensor(last, **i32)}
    return meta, pool, qo[-1], max(total)


def _normal(g, shape, dev, dtype, scale=1.0):
    """Normal values straight into the type, a slice at a time (a cache is large)."""
    out = torch.empty(shape, dtype=dtype, device=dev)
    flat = out.view(-1)
    for a in range(0, flat.numel(), 1 << 28):
        n = min(1 << 28, flat.numel() - a)
        flat[a:a + n] = torch.randn(n, generator=g, device=dev, dtype=torch.float32) * scale
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 2 + 1)
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "logprobs":
        rows, vocab, ld = case["rows"], case["vocab"], case["vocab"] + case["pad"]
        # logits of a trained head: wide, with a few columns that stand out; the columns behind
        # the vocabulary belong to zero rows of a padded head
        logits = _normal(g, (rows, ld), dev, dtype, 2.5)
        if case["pad"]:
            logits[:, vocab:] = 0
        peak = torch.randint(0, vocab, (rows, 3), generator=g, device=dev)
        logits.scatter_(1, peak, (12 + 2 * torch.randn(rows, 3, generator=g, device=dev)).to(dtype))
        if case["masked"]:
            # a grammar allows a part of the vocabulary
            for a in range(0, rows, 64):
                part = logits[a:a + 64, :vocab]
                part.masked_fill_(torch.rand(part.shape, generator=g, device=dev) < 0.5, float("-inf"))
            logits.scatter_(1, peak[:, :1], torch.full((rows, 1), 6.0, device=dev, dtype=dtype))
        tokens = torch.where(torch.rand(rows, generator=g, device=dev) < 0.7, peak[:, 0],
                             torch.randint(0, vocab, (rows,), generator=g, device=dev))
        return dict(case=case, logits=logits, tokens=tokens)
    meta, pool, n_new, longest = _tables(case, g, dev)
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    kc = _normal(g, (pool, case["page"], hkv, dim), dev, dtype)
    vc = _normal(g, (pool, case["page"], hkv, dim), dev, dtype)
    state = dict(case=case, meta=meta, k_cache=kc, v_cache=vc, longest=longest, n_new=n_new)
    if case["op"] == "decode":
        # wide enough that a few positions carry most of the weight
        state["q"] = _normal(g, (case["requests"], hq, dim), dev, dtype, 2.0)
    else:
        group = hq // hkv
        if case["packed"]:                       # rows of a fused projection, per K/V head [q.. | k | v]
            rows = _normal(g, (n_new, hkv, group + 2, dim), dev, dtype)
            state["q"], state["k"], state["v"] = rows[:, :, :group], rows[:, :, group], rows[:, :, group + 1]
        else:
            state["q"] = _normal(g, (n_new, hkv, group, dim), dev, dtype)
            state["k"] = _normal(g, (n_new, hkv, dim), dev, dtype)
            state["v"] = _normal(g, (n_new, hkv, dim), dev, dtype)
        rot = case["rot"]
        freq = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
        ang = torch.arange(longest, dtype=torch.float64, device=dev)[:, None] * freq[None, :]
        ang = torch.cat((ang, ang), dim=1)
        table = _DTYPES[case["table"]]
        state["cos"], state["sin"] = ang.cos().to(table), ang.sin().to(table)
        state["q_norm"] = state["k_norm"] = None
        if case["norm"]:
            state["q_norm"] = _normal(g, (dim,), dev, torch.float32, 0.1).add_(1).to(dtype)
            state["k_norm"] = _normal(g, (dim,), dev, torch.float32, 0.1).add_(1).to(dtype)
    if own:
        # the handle a serving program keeps for each layer of its cache
        import yirage_b200
        state["cache"] = yirage_b200.PagedKVCache(kc, vc, meta)
    return state


# --------------------------------------------------------------------------------- plain form
def _lengths(meta, page):
    indptr = meta["paged_kv_indptr_buffer"].long()
    pages = indptr[1:] - indptr[:-1]
    return torch.where(pages > 0, (pages - 1) * page + meta["paged_kv_last_page_len_buffer"].long(), pages * 0)


def _plain_rotate(x, weight, cos, sin, eps):
    """x [tokens, heads, dim] in 32 bits: RMS norm over dim where a weight is given, then the
    first rot dimensions rotated against the tables [tokens, 1, rot]."""
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + eps) * weight.float()
    rot = cos.shape[-1]
    half = rot // 2
    a, b, rest = x[..., :half], x[..., half:rot], x[..., rot:]
    return torch.cat((a * cos[..., :half] - b * sin[..., :half], b * cos[..., half:] + a * sin[..., half:], rest), dim=-1)


def _plain_append(s):
    case, meta, page = s["case"], s["meta"], s["case"]["page"]
    n = s["n_new"]
    qo = meta["qo_indptr_buffer"].long()
    t = torch.arange(n, device=qo.device)
    req = (t[:, None] >= qo[None, 1:]).sum(dim=1)
    pos = _lengths(meta, page)[req] - (qo[req + 1] - t)
    slot = meta["paged_kv_indices_buffer"].long()[meta["paged_kv_indptr_buffer"].long()[req] + pos // page]
    cos, sin = s["cos"][pos].float()[:, None], s["sin"][pos].float()[:, None]
    q = _plain_rotate(s["q"].float().reshape(n, case["hq"], case["dim"]), s["q_norm"], cos, sin, 1e-6)
    k = _plain_rotate(s["k"].float(), s["k_norm"], cos, sin, 1e-6)
    s["k_cache"][slot, pos % page] = k.to(s["k_cache"].dtype)
    s["v_cache"][slot, pos % page] = s["v"]
    return q.to(s["q"].dtype)


def _plain_decode(s):
    case, meta, page = s["case"], s["meta"], s["case"]["page"]
    hkv, dim, n = case["hkv"], case["dim"], case["requests"]
    length = _lengths(meta, page)
    pos = torch.arange(max(1, s["longest"]), device=length.device)
    at = (meta["paged_kv_indptr_buffer"].long()[:-1, None] + pos[None, :] // page)
    table = meta["paged_kv_indices_buffer"].long()
    slot = table[at.clamp(max=table.numel() - 1)]
    k = s["k_cache"][slot, (pos % page)[None, :]].float()            # [requests, longest, hkv, dim]
    v = s["v_cache"][slot, (pos % page)[None, :]].float()
    q = s["q"].float().view(n, hkv, case["hq"] // hkv, dim)
    score = torch.matmul(q, k.permute(0, 2, 3, 1)) * (dim ** -0.5)
    seen = pos[None, :] < length[:, None]
    if case["window"]:
        seen = seen & (pos[None, :] >= length[:, None] - case["window"])
    score = torch.where(seen[:, None, None, :], score, float("-inf"))
    top = score.amax(dim=-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    weight = torch.exp(score - top)
    total = weight.sum(dim=-1, keepdim=True)
    out = torch.matmul(weight, v.permute(0, 2, 1, 3)) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total))[..., 0]
    return out.reshape(n, case["hq"], dim).to(s["q"].dtype), lse.reshape(n, case["hq"])


def _plain_logprobs(s):
    case = s["case"]
    x = s["logits"][:, :case["vocab"]].float()
    top = x.amax(dim=-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(dim=-1, keepdim=True)
    logp = x - top - torch.log(total)
    entropy = -torch.where(e > 0, e * logp, 0.0).sum(dim=-1) / total[:, 0]
    given = logp.gather(1, s["tokens"][:, None])[:, 0]
    if not case["top"]:
        return given, entropy
    best = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
    return given, entropy, logp.gather(1, best), best


# ---------------------------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    if case["op"] == "append":
        if own:
            q = state["cache"].append(state["k"], state["v"], q=state["q"], cos=state["cos"], sin=state["sin"],
                                      q_norm=state["q_norm"], k_norm=state["k_norm"], eps=1e-6)
        else:
            q = _plain_append(state)
        return q, state["k_cache"], state["v_cache"]
    if case["op"] == "decode":
        if own:
            return state["cache"].decode(state["q"], window=case["window"], return_lse=True)
        return _plain_decode(state)
    if own:
        import yirage_b200
        got = yirage_b200.token_logprobs(state["logits"], state["tokens"], top_k=case["top"],
                                         valid_cols=case["vocab"])
        return tuple(got) if case["top"] else (got.logprob, got.entropy)
    return _plain_logprobs(state)


def work(case):
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * _SIZE[case["dtype"]] + case["rows"] * (8 + 4 + 4 + 12 * case["top"]), "flops": 5 * n}
    ctx, new = _plan(case)
    hq, hkv, dim, size = case["hq"], case["hkv"], case["dim"], _SIZE[case["dtype"]]
    if case["op"] == "append":
        n = sum(new)
        positions = min(n, max(c + m for c, m in zip(ctx, new)))
        return {"bytes": 2 * n * (hq + 2 * hkv) * dim * size + 2 * positions * case["rot"] * _SIZE[case["table"]],
                "flops": n * (hq + hkv) * (3 * case["rot"] + (4 * dim if case["norm"] else 0))}
    seen = sum(min(c, case["window"]) if case["window"] else c for c in ctx)
    return {"bytes": 2 * seen * hkv * dim * size + case["requests"] * hq * (2 * dim * size + 4),
            "flops": 4 * seen * hq * dim}


# -------------------------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "logprobs":
        logits, vocab, k = s["logits"], case["vocab"], case["top"]
        given, entropy, best, ids = [], [], [], []
        column = torch.arange(vocab, device=logits.device)
        for a in range(0, case["rows"], 128):
            x = logits[a:a + 128, :vocab].to(f64)
            lse = torch.logsumexp(x, dim=1)
            p = torch.exp(x - lse[:, None])
            given.append(x[torch.arange(x.shape[0], device=x.device), s["tokens"][a:a + 128]] - lse)
            entropy.append(lse - (p * torch.where(p > 0, x, 0.0)).sum(dim=1))
            if k:
                # one whole number per column: its value's order first, the lower column on ties
                bits = (logits[a:a + 128, :vocab].float() + 0.0).view(torch.int32).long()
                order = torch.where(bits >= 0, bits, -(bits & 0x7fffffff))
                where = torch.topk(order * (1 << 20) - column, k, dim=1).indices
                ids.append(where)
                best.append(x.gather(1, where) - lse[:, None])
        if not k:
            return torch.cat(given), torch.cat(entropy)
        return torch.cat(given), torch.cat(entropy), torch.cat(best), torch.cat(ids)
    meta = {key: value.tolist() for key, value in s["meta"].items()}
    ctx, new = _plan(case)
    page, hq, hkv, dim = case["page"], case["hq"], case["hkv"], case["dim"]
    dev = s["k_cache"].device
    q_all, lse_all = [], []
    if case["op"] == "append":
        kc, vc = s["k_cache"].to(f64), s["v_cache"].to(f64)
        rot = case["rot"]
        swap = torch.cat((torch.arange(rot // 2, rot), torch.arange(rot // 2))).to(dev)
        sign = torch.cat((-torch.ones(rot // 2), torch.ones(rot // 2))).to(dev, f64)
    for r in range(case["requests"]):
        where = meta["paged_kv_indices_buffer"][meta["paged_kv_indptr_buffer"][r]:meta["paged_kv_indptr_buffer"][r + 1]]
        first = meta["qo_indptr_buffer"][r]
        total = ctx[r] + new[r]
        pages = torch.tensor(where, dtype=torch.long, device=dev)
        if case["op"] == "append":
            pos = torch.arange(ctx[r], total, device=dev)
            rows = slice(first, first + new[r])
            done = []
            for x, w in ((s["q"][rows].to(f64).reshape(new[r], hq, dim), s["q_norm"]), (s["k"][rows].to(f64), s["k_norm"])):
                if w is not None:
                    x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / dim + 1e-6) * w.to(f64)
                head = x[..., :rot]
                turned = head * s["cos"].to(f64)[pos][:, None] + head[..., swap] * sign * s["sin"].to(f64)[pos][:, None]
                done.append(torch.cat((turned, x[..., rot:]), dim=-1))
            q_all.append(done[0])
            kc[pages[pos // page], pos % page] = done[1]
            vc[pages[pos // page], pos % page] = s["v"][rows].to(f64)
            continue
        lo = max(0, total - case["window"]) if case["window"] else 0
        if total == 0:
            q_all.append(torch.zeros(hq, dim, dtype=f64, device=dev))
            lse_all.append(torch.full((hq,), float("-inf"), dtype=f64, device=dev))
            continue
        pos = torch.arange(lo, total, device=dev)
        k = s["k_cache"][pages[pos // page], pos % page].to(f64)
        v = s["v_cache"][pages[pos // page], pos % page].to(f64)
        q = s["q"][r].to(f64).view(hkv, hq // hkv, dim)
        score = torch.einsum("hgd,phd->hgp", q, k) / math.sqrt(dim)
        q_all.append(torch.einsum("hgp,phd->hgd", torch.softmax(score, dim=-1), v).reshape(hq, dim))
        lse_all.append(torch.logsumexp(score, dim=-1).reshape(hq))
    if case["op"] == "append":
        return torch.cat(q_all), kc, vc
    return torch.stack(q_all), torch.stack(lse_all)
