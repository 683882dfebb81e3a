"""Cases for the target model's side of a speculation round: attention of the
new tokens over a paged key-value cache, eviction from that cache by
accumulated attention weight, and verification of the drafted tokens.

``listed()`` and ``draw()`` give cases, ``prepare()`` makes a case's inputs on
the GPU from a seed, ``run()`` makes one pass (the plain torch form, or with
``own`` set the library's operators), ``work()`` counts the bytes and
operations no implementation can do without, and ``exact()`` computes the
same outputs in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# chance that a drafted token is accepted with the logits that prepare() makes
AGREE = 0.75


def _attention(name, batch, q_heads, kv_heads, head_dim, new, min_len, max_len, page, dtype="bf16", window=0, sinks=0,
               append=False, weights=False):
    return {"name": name, "op": "attention", "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "new": new, "min_len": min_len, "max_len": max_len, "page": page, "dtype": dtype,
            "window": window, "sinks": sinks, "append": append, "weights": weights}


def _evict(name, batch, kv_heads, head_dim, min_len, max_len, page, keep, recent, first, dtype="bf16"):
    return {"name": name, "op": "evict", "batch": batch, "kv_heads": kv_heads, "head_dim": head_dim,
            "min_len": min_len, "max_len": max_len, "page": page, "keep": keep, "recent": recent, "first": first,
            "dtype": dtype}


def _verify(name, batch, draft, vocab, temperature, dtype="bf16"):
    return {"name": name, "op": "verify", "batch": batch, "draft": draft, "vocab": vocab, "temperature": temperature,
            "dtype": dtype}


def listed():
    return [
        # one chat: a token is appended and attends to 1K tokens; latency is all there is
        _attention("attn_1x1k", 1, 12, 2, 128, 1, 1024, 1024, 16, append=True),
        # one long document, 32K tokens: a single row of work split over the whole GPU
        _attention("attn_1x32k", 1, 12, 2, 128, 1, 32768, 32768, 64),
        # a serving batch of very unequal lengths, fp16, each step with its append
        _attention("attn_32_ragged", 32, 32, 8, 64, 1, 1, 8192, 16, "fp16", append=True),
        # verification: the last accepted token and four drafted ones attend at once
        _attention("attn_64_new5", 64, 12, 2, 128, 5, 4000, 16384, 32),
        # long contexts at the full head count: the most bytes of all
        _attention("attn_16_long", 16, 32, 8, 128, 1, 16384, 32768, 64),
        # short window and sinks over a large batch of short chats
        _attention("window_128", 128, 12, 2, 128, 1, 1, 4096, 16, window=1024, sinks=4, append=True),
        # long window, verification of three drafted tokens, pages that end inside every tile
        _attention("window_8_new4", 8, 32, 8, 64, 4, 20000, 32768, 24, window=4095, sinks=5),
        # a step of a cache that is to be evicted from: attention weights are added up
        _attention("attn_16_weights", 16, 12, 2, 128, 1, 1000, 8192, 16, weights=True),
        # one sequence over its budget
        _evict("evict_1x5k", 1, 2, 128, 5000, 5000, 16, 1024, 256, 4),
        # a batch brought back to its budget at once
        _evict("evict_32", 32, 8, 64, 4096, 16384, 32, 4096, 1024, 4),
        # greedy decoding of a small batch
        _verify("verify_4_greedy", 4, 4, 32000, 0.0),
        # sampling for a serving batch over a large vocabulary
        _verify("verify_64", 64, 5, 128000, 0.8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["attention", "attention", "attention", "evict", "verify"])
    if op == "verify":
        batch, draft, vocab = _log(rng, 1, 96), rng.randint(1, 8), _log(rng, 1000, 160000)
        if rng.random() < 0.5:
            vocab = vocab // 64 * 64
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        batch = max(1, min(batch, 60_000_000 // ((2 * draft + 1) * vocab * (2 if dtype == "fp32" else 1))))
        c = _verify("", batch, draft, vocab, rng.choice([0.0, 0.6, 1.0, 1.3]), dtype)
    elif op == "evict":
        batch, (kv_heads, head_dim) = _log(rng, 1, 48), rng.choice([(2, 128), (8, 64), (8, 128), (1, 128), (4, 64)])
        max_len = _log(rng, 300, 40000)
        keep = max(16, int(max_len * rng.uniform(0.1, 0.7)))
        batch = max(1, min(batch, 400_000_000 // (max_len * kv_heads * head_dim * 4)))
        c = _evict("", batch, kv_heads, head_dim, max(1, int(max_len * rng.uniform(0.05, 1.0))), max_len,
                   rng.choice([8, 16, 20, 32, 64]), keep, int(keep * rng.uniform(0.0, 0.6)), rng.randint(0, 8),
                   rng.choice(["bf16", "fp16"]))
    else:
        batch = _log(rng, 1, 128)
        q_heads, kv_heads, head_dim = rng.choice([(12, 2, 128), (32, 8, 64), (32, 8, 128), (6, 2, 128), (8, 8, 64),
                                                  (16, 1, 128), (14, 2, 64)])
        new = rng.choice([1, 1, 1, 2, 3, 4, 5, 8])
        max_len = _log(rng, 16, 32768)
        min_len = max(1, int(max_len * rng.uniform(0.0, 1.0)))
        batch = max(1, min(batch, 1_000_000_000 // (max_len * kv_heads * head_dim * 4),
                           700_000_000 // (max_len * q_heads * new)))
        window = rng.choice([0, 0, _log(rng, 1, 8192)])
        c = _attention("", batch, q_heads, kv_heads, head_dim, new, min_len, max_len, rng.choice([8, 16, 16, 24, 32, 64]),
                       rng.choice(["bf16", "bf16", "fp16"]), window, rng.randint(0, 8) if window else 0,
                       rng.random() < 0.3, rng.random() < 0.25)
    del c["name"]
    return c


# ------------------------------------------------------------------- inputs
def _lengths(case):
    """The batch's lengths, evenly spread; the seed only orders them."""
    n = case["batch"]
    if n == 1:
        return [case["max_len"]]
    return [case["min_len"] + (case["max_len"] - case["min_len"]) * i // (n - 1) for i in range(n)]


def _pool(case, lengths, more, gen):
    """Key and value pages, and a block table [batch, M] of shuffled page
    numbers (-1 where a sequence has no page); `more`: spare pages."""
    page, dtype = case["page"], DTYPES[case["dtype"]]
    need = [-(-n // page) for n in lengths]
    total = sum(need) + more
    shape = (total, case["kv_heads"], page, case["head_dim"])
    k = torch.randn(shape, device="cuda", generator=gen).to(dtype)
    v = torch.randn(shape, device="cuda", generator=gen).to(dtype)
    k[..., torch.randperm(case["head_dim"], device="cuda", generator=gen)[:4]] *= 8   # channels that stand out
    order = torch.randperm(total, device="cuda", generator=gen)
    table = torch.full((case["batch"], -(-case["max_len"] // page) + 2), -1, dtype=torch.int64)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(at, at + n)
        at += n
    table = table.cuda()
    return k, v, torch.where(table >= 0, order[table.clamp_min(0)], table).to(torch.int32), order[at:]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "verify":
        B, K, V = case["batch"], case["draft"], case["vocab"]
        dtype, temp = DTYPES[case["dtype"]], case["temperature"]
        target = torch.randn(B, K + 1, V, device="cuda", generator=gen).mul_(2.0)
        at = torch.randint(V, (B, K + 1, 16), device="cuda", generator=gen)     # a few likely continuations
        target.scatter_add_(2, at, 6 + 8 * torch.rand(at.shape, device="cuda", generator=gen))
        draft = target[:, :K] + 0.7 * torch.randn(B, K, V, device="cuda", generator=gen)
        target, draft = target.to(dtype), draft.to(dtype)
        if temp > 0:
            e = torch.empty(B, K, V, device="cuda").exponential_(generator=gen)
            tokens = (torch.softmax(draft.float() / temp, -1) / e).argmax(-1)
        else:
            tokens = draft.argmax(-1)
        return {"case": case, "target": target, "draft": draft, "tokens": tokens,
                "uniforms": torch.rand(B, K, device="cuda", generator=gen),
                "noise": torch.empty(B, V, device="cuda").exponential_(generator=gen).clamp_min_(1e-30)}
    lengths = _lengths(case)
    at = torch.randperm(len(lengths), device="cuda", generator=gen).tolist()
    lengths = [lengths[i] for i in at]
    if case["op"] == "evict":
        page, B = case["page"], case["batch"]
        kept_pages = -(-case["keep"] // page)
        k, v, table, spare = _pool(case, lengths, B * kept_pages, gen)
        weights = torch.empty(B, table.shape[1] * page, device="cuda").exponential_(generator=gen).pow_(3)
        return {"case": case, "k": k, "v": v, "table": table, "lengths": torch.tensor(lengths, dtype=torch.int32).cuda(),
                "weights": weights, "new_table": spare.view(B, kept_pages).to(torch.int32)}
    k, v, table, _ = _pool(case, lengths, 3, gen)
    B, T, D, dtype = case["batch"], case["new"], case["head_dim"], DTYPES[case["dtype"]]
    s = {"case": case, "k": k, "v": v, "table": table, "lengths": torch.tensor(lengths, dtype=torch.int32).cuda(),
         # as a projection leaves it: [batch, new, heads, head_dim], seen with the heads first
         "q": torch.randn(B, T, case["q_heads"], D, device="cuda", generator=gen).to(dtype).transpose(1, 2)}
    if case["append"]:
        s["k_new"] = torch.randn(B, T, case["kv_heads"], D, device="cuda", generator=gen).to(dtype).transpose(1, 2)
        s["v_new"] = torch.randn(B, T, case["kv_heads"], D, device="cuda", generator=gen).to(dtype).transpose(1, 2)
    if case["weights"]:
        s["weights"] = torch.rand(B, table.shape[1] * case["page"], device="cuda", generator=gen)
    return s


# --------------------------------------------------------------------- runs
def run(state):
    return {"attention": _run_attention, "evict": _run_evict, "verify": _run_verify}[state["case"]["op"]](state)


def _run_attention(s):
    c = s["case"]
    if own:
        import kv_reduce_b200 as kvr

        if c["append"]:
            kvr.paged_append(s["k_new"], s["v_new"], s["k"], s["v"], s["table"], s["lengths"])
        out = kvr.paged_decode_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], window=c["window"],
                                         sinks=c["sinks"], token_weights=s.get("weights"))
    else:
        B, T, HQ, H, D, page = c["batch"], c["new"], c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
        lengths = s["lengths"].long()
        if c["append"]:
            pos = lengths[:, None] - T + torch.arange(T, device="cuda")                # [B, T]
            fits = pos >= 0                                                            # a sequence shorter than T
            pages = s["table"].long().gather(1, (pos // page).clamp_min(0))
            where = (pages[fits], slice(None), (pos % page)[fits])
            s["k"][where] = s["k_new"].transpose(1, 2)[fits]
            s["v"][where] = s["v_new"].transpose(1, 2)[fits]
        table = s["table"].long().clamp_min(0)
        n = table.shape[1] * page
        keys = s["k"][table].transpose(1, 2).reshape(B, H, n, D).float()
        values = s["v"][table].transpose(1, 2).reshape(B, H, n, D).float()
        j = torch.arange(n, device="cuda")
        values = torch.where((j < lengths[:, None])[:, None, :, None], values, 0.0)
        i = lengths[:, None] - T + torch.arange(T, device="cuda")                      # [B, T]
        seen = j <= i[..., None]                                                       # [B, T, n]
        if c["window"]:
            seen &= (j > i[..., None] - c["window"]) | (j < c["sinks"])
        seen = seen[:, None, None]                                                     # [B, 1, 1, T, n]
        q = s["q"].float().reshape(B, H, HQ // H * T, D)
        scores = (q @ keys.transpose(2, 3)).view(B, H, HQ // H, T, n) / math.sqrt(D)
        scores = torch.where(seen, scores, -math.inf)
        top = scores.amax(-1, keepdim=True)
        p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
        out = (p.view(B, H, HQ // H * T, n) @ values).view(B, HQ, T, D).to(s["q"].dtype)
        if c["weights"]:
            s["weights"] += p.sum((1, 2, 3))
    got = {"out": out}
    if c["append"]:
        got |= {"key_pages": s["k"], "value_pages": s["v"]}
    if c["weights"]:
        got["weights"] = s["weights"]
    return got


def _run_evict(s):
    c = s["case"]
    if own:
        import kv_reduce_b200 as kvr

        kept, lengths, weights = kvr.paged_evict(s["k"], s["v"], s["table"], s["lengths"], s["weights"], s["new_table"],
                                                 keep=c["keep"], recent=c["recent"], first=c["first"])
    else:
        page, keep = c["page"], c["keep"]
        old = s["lengths"].long()[:, None]                                             # [B, 1]
        n = max(s["weights"].shape[1], keep)
        w = torch.nn.functional.pad(s["weights"], (0, n - s["weights"].shape[1]))
        j = torch.arange(n, device="cuda")
        always = (j < c["first"]) | (j >= old - c["recent"]) | (old <= keep)
        rank = torch.where(always, math.inf, w)
        rank = torch.where(j < old, rank, -math.inf)
        order = rank.sort(dim=1, descending=True, stable=True).indices[:, :keep]           # ties: the lowest index first
        lengths = old.clamp_max(keep)
        slot = torch.arange(keep, device="cuda")
        live = slot < lengths
        kept = torch.where(live, order, n).sort(1).values
        src = torch.where(live, kept, 0)
        weights = torch.where(live, w.gather(1, src), 0.0)
        src_page = s["table"].long().gather(1, src // page)
        dst_page = s["new_table"].long()[:, slot // page].expand(len(old), -1)
        for pool in (s["k"], s["v"]):
            rows = pool[src_page[live], :, (src % page)[live]]
            pool[dst_page[live], :, (slot % page).expand(len(old), -1)[live]] = rows
        kept = torch.where(live, kept, -1).to(torch.int32)
        lengths = lengths[:, 0].to(torch.int32)
    return {"kept": kept, "lengths": lengths, "weights": weights, "key_pages": s["k"], "value_pages": s["v"]}


def _run_verify(s):
    c = s["case"]
    if own:
        import kv_reduce_b200 as kvr

        r = kvr.verify_draft_tokens(s["target"], s["draft"], s["tokens"], s["uniforms"], s["noise"],
                                    temperature=c["temperature"])
        return {"tokens": r.tokens, "accepted": r.accepted, "accept_prob": r.accept_prob}
    B, K, temp = c["batch"], c["draft"], c["temperature"]
    slot = torch.arange(K + 1, device="cuda")
    if temp == 0:
        best = s["target"].max(-1).indices if s["target"].dtype == torch.float32 else s["target"].float().max(-1).indices
        prob = (s["tokens"] == best[:, :K]).float()
        taken = prob > 0
    else:
        lt = s["target"][:, :K].float() / temp
        ld = s["draft"].float() / temp
        mt, md = lt.amax(-1, keepdim=True), ld.amax(-1, keepdim=True)
        zt = torch.exp(lt - mt).sum(-1, keepdim=True)
        zd = torch.exp(ld - md).sum(-1, keepdim=True)
        x = s["tokens"][..., None]
        ratio = torch.exp((lt.gather(2, x) - mt) - (ld.gather(2, x) - md)) * (zd / zt)
        prob = ratio[..., 0].clamp_max(1.0)
        taken = s["uniforms"] < prob
    run_of = taken.long().cumprod(1)
    accepted = run_of.sum(1)                                                           # [B]
    at = accepted[:, None]
    if temp == 0:
        last = best.gather(1, at)[:, 0]
    else:
        rows = torch.arange(B, device="cuda")
        lj = s["target"][rows, accepted].float() / temp
        p = torch.exp(lj - lj.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        j = accepted.clamp_max(K - 1)
        q = torch.exp(ld[rows, j] - md[rows, j]) / zd[rows, j]
        q = torch.where(at < K, q, 0.0)
        rest = (p - q).clamp_min(0.0)
        rest = torch.where((rest > 0).any(-1, keepdim=True), rest, p)
        last = (rest / s["noise"]).max(-1).indices
    drafted = torch.nn.functional.pad(s["tokens"], (0, 1))
    tokens = torch.where(slot < at, drafted, torch.where(slot == at, last[:, None], -1))
    prob = torch.where(slot[:K] <= at, prob, 0.0)
    return {"tokens": tokens, "accepted": accepted.to(torch.int32), "accept_prob": prob}


# --------------------------------------------------------------------- work
def work(case):
    if case["op"] == "verify":
        B, K, V = case["batch"], case["draft"], case["vocab"]
        size = 4 if case["dtype"] == "fp32" else 2
        looked_at = sum(AGREE ** k for k in range(K))      # positions up to the first refusal, on average
        last = AGREE ** K                                  # the row after the last drafted token
        if case["temperature"] == 0:
            rows, noise = looked_at + last, 0
        else:
            rows, noise = 2 * looked_at + last, 4 * V
        return {"bytes": B * (rows * V * size + noise + (K + 1) * 24), "flops": B * rows * V * 4}
    lengths, D, H = _lengths(case), case["head_dim"], case["kv_heads"]
    if case["op"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lengths)
        return {"bytes": 4 * sum(lengths) + kept * (H * D * 8 + 8), "flops": sum(lengths)}
    T, HQ, window = case["new"], case["q_heads"], case["window"]
    seen = sum(min(n, case["sinks"] + window + T - 1) if window else n for n in lengths)
    q = len(lengths) * T * HQ * D * 2
    extra = (len(lengths) * T * H * D * 8 if case["append"] else 0) + (8 * seen if case["weights"] else 0)
    return {"bytes": seen * H * D * 4 + 2 * q + extra, "flops": 4 * D * HQ * T * seen}


# -------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "evict": _exact_evict, "verify": _exact_verify}[case["op"]](s)


def _exact_attention(s):
    c = s["case"]
    T, HQ, H, D, page = c["new"], c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    k, v = s["k"], s["v"]
    outs = []
    for b, n in enumerate(s["lengths"].tolist()):
        rows = torch.arange(n, device="cuda")
        pages, inside = s["table"][b, rows // page].long(), rows % page
        if c["append"]:
            new = min(T, n)
            k[pages[n - new:], :, inside[n - new:]] = s["k_new"][b, :, T - new:].transpose(0, 1)
            v[pages[n - new:], :, inside[n - new:]] = s["v_new"][b, :, T - new:].transpose(0, 1)
        keys, values = k[pages, :, inside].double(), v[pages, :, inside].double()      # [n, H, D]
        out = torch.zeros(HQ, T, D, dtype=torch.float64, device="cuda")
        for t in range(T):
            i = n - T + t
            if i < 0:
                continue
            lo = max(0, i - c["window"] + 1) if c["window"] else 0
            at = torch.cat([rows[:min(c["sinks"], lo)], rows[lo:i + 1]])
            q = s["q"][b, :, t].double().view(H, HQ // H, D)
            p = torch.softmax(torch.einsum("hgd,nhd->hgn", q, keys[at]) * D ** -0.5, -1)
            out[:, t] = torch.einsum("hgn,nhd->hgd", p, values[at]).reshape(HQ, D)
            if c["weights"]:
                if "total" not in s:
                    s["total"] = s["weights"].double()
                s["total"][b, at] += p.sum((0, 1))
        outs.append(out)
    got = {"out": torch.stack(outs)}
    if c["append"]:
        got |= {"key_pages": k.double(), "value_pages": v.double()}
    if c["weights"]:
        got["weights"] = s.get("total", s["weights"].double())
    return got


def _exact_evict(s):
    c = s["case"]
    page, keep, k, v = c["page"], c["keep"], s["k"], s["v"]
    weights = torch.zeros(len(s["lengths"]), keep, dtype=torch.float64)
    for b, n in enumerate(s["lengths"].tolist()):
        w = s["weights"][b, :n].tolist()
        kept = list(range(n))
        if n > keep:
            forced = [j for j in kept if j < c["first"] or j >= n - c["recent"]]
            others = sorted(set(kept) - set(forced), key=lambda j: (-w[j], j))
            kept = sorted(forced + others[:keep - len(forced)])
        weights[b, :len(kept)] = torch.tensor([w[j] for j in kept], dtype=torch.float64)
        src, dst = torch.tensor(kept, device="cuda"), torch.arange(len(kept), device="cuda")
        for pool in (k, v):
            pool[s["new_table"][b, dst // page].long(), :, dst % page] = pool[s["table"][b, src // page].long(), :,
                                                                              src % page]
    return {"kept": None, "lengths": None, "weights": weights, "key_pages": k.double(), "value_pages": v.double()}


def _exact_verify(s):
    c = s["case"]
    B, K, temp = c["batch"], c["draft"], c["temperature"]
    prob = torch.zeros(B, K, dtype=torch.float64)
    for b in range(B):
        for j in range(K):
            x = int(s["tokens"][b, j])
            if temp == 0:
                row = s["target"][b, j]
                prob[b, j] = float(x == int((row == row.max()).nonzero()[0, 0]))
                stop = prob[b, j] == 0
            else:
                lp = torch.log_softmax(s["target"][b, j].double() / temp, -1)[x]
                lq = torch.log_softmax(s["draft"][b, j].double() / temp, -1)[x]
                prob[b, j] = min(1.0, math.exp(float(lp - lq)))
                stop = not float(s["uniforms"][b, j]) < prob[b, j]
            if stop:
                break
    return {"tokens": None, "accepted": None, "accept_prob": prob}
