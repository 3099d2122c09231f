"""The serving path's operators for long conversations, as measured cases: attention with a sliding window and
sink positions, copies of cache pages, and log probabilities of tokens.

`run` computes an operator in elementary torch operations where `own` is false and through `accel_b200.tensor`
where it is true.  `exact` restates each operator in 64 bits."""
import math

import torch

own = False

DEV = "cuda"
F16 = "f16"


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one conversation, a short window: the smallest call a decode loop makes, where latency counts
        dict(name="decode_one", op="decode", batch=1, kv=8, group=4, dim=128, block=16, window=256, sinks=4,
             len_min=1000, len_max=1000, cache="f32"),
        # the benchmark's batch (32 heads over an f32 cache), a window of 1024 behind a context of 2048
        dict(name="decode_batch", op="decode", batch=16, kv=32, group=1, dim=128, block=16, window=1024, sinks=4,
             len_min=2048, len_max=2048, cache="f32"),
        # grouped heads over an f16 cache, long ragged conversations whose far pages have been freed
        dict(name="decode_grouped_f16", op="decode", batch=32, kv=8, group=4, dim=128, block=16, window=4096, sinks=16,
             len_min=3000, len_max=40000, cache=F16),
        # odd everything: head dimension, group, page size, window, sinks; lengths from one token on
        dict(name="decode_odd", op="decode", batch=7, kv=5, group=3, dim=40, block=13, window=777, sinks=3,
             len_min=1, len_max=1500, cache="f32"),
        # one scheduler step of several sequences: prompts' chunks beside single tokens
        dict(name="ragged_step", op="ragged", batch=12, kv=8, group=4, dim=128, block=16, window=1024, sinks=4,
             len_min=300, len_max=3000, chunk=64, cache=F16),
        # a chunk of a prompt behind a long context
        dict(name="prefill_chunk", op="prefill", tokens=256, base=1801, kv=8, group=4, dim=128, block=16, window=1024,
             sinks=4, paged=True, cache="f32"),
        # a long prompt, grouped heads, f16 cache
        dict(name="prefill_grouped_f16", op="prefill", tokens=4096, base=0, kv=8, group=4, dim=128, block=16,
             window=2048, sinks=4, paged=True, cache=F16),
        # the largest: a prompt's second half, every head with a cache of its own
        dict(name="prefill_long", op="prefill", tokens=4096, base=4096, kv=32, group=1, dim=128, block=16, window=4096,
             sinks=8, paged=False, cache="f32"),
        # a fork's copy on write: the last, partly filled page of one sequence in every cache of a small model
        dict(name="pages_fork", op="pages", caches=8, pages=64, pairs=1, block=16, kv=8, dim=128, cache=F16),
        # compaction: a quarter of a pool's pages move
        dict(name="pages_compact", op="pages", caches=16, pages=256, pairs=64, block=16, kv=32, dim=128, cache="f32"),
        # a decode step's sampled tokens with five alternatives each
        dict(name="logprobs_step", op="logprobs", rows=16, vocab=32000, targets=1, top=5, masked=0, logits="f32"),
        # a scored prompt: every token's log probability, entropy and twenty alternatives
        dict(name="logprobs_prompt", op="logprobs", rows=2048, vocab=32000, targets=1, top=20, masked=0, logits="f32"),
    ]


def _log(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "ragged", "prefill", "prefill", "pages", "logprobs", "logprobs"])
    cache = rng.choice(["f32", F16])
    kv, group, dim = rng.choice([1, 2, 4, 5, 8, 16, 32]), rng.choice([1, 2, 3, 4, 6, 8]), rng.choice([40, 64, 80, 96, 128, 128])
    if kv * group > 64:
        group = 1
    head = dict(kv=kv, group=group, dim=dim, block=rng.choice([1, 8, 13, 16, 16, 32]),
                window=_log(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 7, 16, 64]), cache=cache)
    if op == "decode":
        hi = _log(rng, 40, 30000)
        c = dict(op=op, batch=_log(rng, 1, 48), len_min=max(1, hi // rng.choice([1, 3, 20])), len_max=hi, **head)
        while c["batch"] * (c["window"] + 64) * kv * dim > 1 << 28:
            c["batch"] = max(1, c["batch"] // 2)
        return c
    if op == "ragged":
        hi = _log(rng, 100, 6000)
        c = dict(op=op, batch=_log(rng, 1, 16), len_min=max(80, hi // 4), len_max=max(80, hi), chunk=rng.choice([1, 5, 33, 64]), **head)
        c["window"] = min(c["window"], 1500)
        return c
    if op == "prefill":
        c = dict(op=op, tokens=_log(rng, 1, 3000), base=rng.choice([0, rng.randint(1, 6000)]), paged=rng.random() < 0.6, **head)
        if kv * group > 32:
            c["group"] = 1
        return c
    if op == "pages":
        pages = _log(rng, 8, 512)
        c = dict(op=op, caches=rng.choice([1, 2, 6, 16, 32]), pages=pages, pairs=_log(rng, 1, pages // 2),
                 block=head["block"], kv=kv, dim=dim, cache=cache)
        while c["caches"] * pages * c["block"] * kv * dim > 1 << 28:
            c["caches"], c["kv"] = max(1, c["caches"] // 2), max(1, c["kv"] // 2)
            kv = c["kv"]
            if c["caches"] * pages * c["block"] * kv * dim > 1 << 28:
                c["block"] = max(1, c["block"] // 2)
        return c
    vocab = rng.choice([_log(rng, 300, 150000), 32000, 131072])
    return dict(op=op, rows=_log(rng, 1, max(1, min(3000, (1 << 26) // vocab))), vocab=vocab, targets=rng.choice([1, 1, 4]),
                top=rng.choice([0, 1, 5, 20, 32]), masked=rng.choice([0, 0, 10]), logits=rng.choice(["f32", F16]))


def _dtype(name):
    return torch.float16 if name == F16 else torch.float32


def _lengths(c):
    """A length per sequence, spread over [len_min, len_max]; of the case alone."""
    span = c["len_max"] - c["len_min"] + 1
    return [c["len_min"] + (7919 * (b + 1) * (b + 3)) % span for b in range(c["batch"])]


def _counts(c):
    """Query tokens per sequence of a ragged step: every third a chunk of a prompt, the others one token."""
    return [min(c["chunk"], n) if b % 3 == 0 else 1 for b, n in enumerate(_lengths(c))]


def _row_positions(c):
    """(sequence, position) of every query row, and the sequences' lengths; host numbers."""
    if c["op"] == "decode":
        ln = _lengths(c)
        return [(b, n - 1) for b, n in enumerate(ln)], ln
    if c["op"] == "ragged":
        ln = _lengths(c)
        return [(b, n - m + i) for b, (n, m) in enumerate(zip(ln, _counts(c))) for i in range(m)], ln
    return [(0, c["base"] + i) for i in range(c["tokens"])], [c["base"] + c["tokens"]]


def _visible(p, c):
    lo = max(p + 1 - c["window"], 0)
    return min(c["sinks"], lo) + p + 1 - lo


def work(case):
    c = case
    e = 2 if c.get("cache", c.get("logits")) == F16 else 4
    if c["op"] == "pages":
        return {"bytes": 2 * c["pairs"] * c["caches"] * c["block"] * c["kv"] * c["dim"] * e + 8 * c["pairs"], "flops": 0}
    if c["op"] == "logprobs":
        r = c["rows"]
        return {"bytes": r * c["vocab"] * e + 8 * r * c["targets"] + 4 * r + 8 * r * c["top"], "flops": 4 * r * c["vocab"]}
    rows, ln = _row_positions(c)
    first = {}
    for b, p in rows:
        first[b] = min(p, first.get(b, p))
    union = 0
    for b, p in first.items():
        lo = max(p + 1 - c["window"], 0)
        union += min(c["sinks"], lo) + ln[b] - lo
    heads = c["kv"] * c["group"]
    return {"bytes": 2 * union * c["kv"] * c["dim"] * e + 8 * len(rows) * heads * c["dim"],
            "flops": 4 * heads * c["dim"] * sum(_visible(p, c) for _, p in rows)}


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def prepare(case, seed):
    c, g = case, _generator(seed)
    randn = lambda *s: torch.randn(s, generator=g, device=DEV)
    s = dict(c)
    if c["op"] == "pages":
        # two caches (keys, values) per layer, one tensor each in a user's hands; here views of one
        s["all"] = randn(c["caches"], c["pages"] * c["block"], c["kv"], c["dim"]).to(_dtype(c["cache"]))
        s["list"] = list(s["all"].unbind(0))
        order = torch.randperm(c["pages"], generator=torch.Generator().manual_seed(seed)).tolist()
        s["src"], s["dst"] = order[:c["pairs"]], order[c["pairs"]:2 * c["pairs"]]
        return s
    if c["op"] == "logprobs":
        x = randn(c["rows"], c["vocab"]) * 2.5
        x[:, :: max(1, c["vocab"] // 37)] += 4.0              # a few plausible tokens above the rest
        if c["masked"]:                                       # a grammar's or a vocabulary's padding mask
            x[:, c["masked"]::c["masked"]] = -math.inf
        s["x"] = x.to(_dtype(c["logits"]))
        t = torch.randint(0, c["vocab"], (c["rows"], c["targets"]), generator=g, device=DEV, dtype=torch.int32)
        if c["masked"]:
            t -= (t % c["masked"] == 0).int() * (t > 0).int()
        s["t"] = t[:, 0].contiguous() if c["targets"] == 1 else t
        return s
    rows, ln = _row_positions(c)
    batch, blk, heads = len(ln), c["block"], c["kv"] * c["group"]
    dt = _dtype(c["cache"])
    s["q"] = randn(len(rows), heads, c["dim"]) * 1.5
    s["scale"] = 1.0 / math.sqrt(c["dim"])
    s["lengths"] = torch.tensor(ln, dtype=torch.int32, device=DEV)
    if c["op"] == "prefill" and not c["paged"]:
        s["k"], s["v"] = (randn(ln[0], c["kv"], c["dim"]).to(dt) for _ in range(2))
        return s
    # the pages a serving process still holds: the sinks' and the window's; the freed ones' entries are -1
    oldest = {}
    for b, p in rows:
        oldest[b] = min(p, oldest.get(b, p))
    most = max((n + blk - 1) // blk for n in ln)
    table = torch.full((batch, most), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(ln):
        lo = max(oldest[b] + 1 - c["window"], 0)
        live = torch.zeros((n + blk - 1) // blk, dtype=torch.bool)
        live[lo // blk:] = True
        live[: (min(c["sinks"], lo) + blk - 1) // blk] = True
        k = int(live.sum())
        table[b, : live.numel()][live] = torch.arange(at, at + k, dtype=torch.int32)
        at += k
    pool = at + 3
    perm = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.where(table < 0, table, perm[table.clamp(min=0).long()])
    s["pages"] = table[0].to(DEV) if c["op"] == "prefill" else table.to(DEV)
    s["k"], s["v"] = (randn(pool * blk, c["kv"], c["dim"]).to(dt) for _ in range(2))
    if c["op"] == "ragged":
        s["counts"] = torch.tensor(_counts(c), dtype=torch.int32, device=DEV)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _softmax_times(scores, mask, v):
    """softmax over the last axis of the masked scores, times v; f32."""
    scores = scores.masked_fill(~mask, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return torch.matmul(p, v) / p.sum(-1, keepdim=True)


def _plain_rows(s, pages, pos):
    """Rows with a page row and a position each (a decode step, a ragged step)."""
    rows, blk = pos.numel(), s["block"]
    n = min(s["window"] + s["sinks"], pages.shape[1] * blk)
    lo = (pos + 1 - s["window"]).clamp(min=0)[:, None]
    ns = lo.clamp(max=s["sinks"])
    i = torch.arange(n, device=DEV)[None, :]
    at = torch.where(i < ns, i, i - ns + lo)
    seen = at <= pos[:, None]
    at = torch.where(seen, at, pos[:, None])
    phys = pages.long().gather(1, at // blk) * blk + at % blk
    k = s["k"][phys].float().permute(0, 2, 3, 1)                 # [rows, kv, dim, n]
    q = s["q"].view(rows, s["kv"], s["group"], s["dim"])
    scores = torch.matmul(q, k) * s["scale"]
    out = _softmax_times(scores, seen[:, None, None, :], s["v"][phys].float().transpose(1, 2))
    return out.reshape(rows, -1, s["dim"])


def _plain_prefill(s):
    t, base, blk = s["tokens"], s["base"], s["block"]
    lo = max(base + 1 - s["window"], 0)
    at = torch.cat([torch.arange(min(s["sinks"], lo), device=DEV), torch.arange(lo, base + t, device=DEV)])
    phys = s["pages"].long()[at // blk] * blk + at % blk if s["paged"] else at
    k, v = (s[x][phys].float().transpose(0, 1) for x in "kv")    # [kv, n, dim]
    q = s["q"].view(t, s["kv"], s["group"], s["dim"]).permute(1, 2, 0, 3)
    pos = base + torch.arange(t, device=DEV)[:, None]
    seen = (at <= pos) & ((at > pos - s["window"]) | (at < s["sinks"]))
    scores = torch.matmul(q, k[:, None].transpose(2, 3)) * s["scale"]
    out = _softmax_times(scores, seen, v[:, None])
    return out.permute(2, 0, 1, 3).reshape(t, -1, s["dim"])


def _plain_logprobs(s):
    x = s["x"].float()
    d = x - x.amax(1, keepdim=True)
    e = torch.exp(d)
    z = e.sum(1, keepdim=True)
    log_z = torch.log(z)
    entropy = log_z[:, 0] - torch.where(e > 0, d * e, 0.0).sum(1) / z[:, 0]
    lp = d - log_z
    t = s["t"].long().view(s["rows"], -1)
    out = {"logprobs": lp.gather(1, t).view(s["t"].shape), "entropy": entropy}
    if s["top"]:
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :s["top"]]
        out["top_ids"], out["top_logprobs"] = ids.int(), lp.gather(1, ids)
    return out


def run(state):
    s = state
    if own:
        return _own(s)
    if s["op"] == "decode":
        return _plain_rows(s, s["pages"], s["lengths"].long() - 1)
    if s["op"] == "ragged":
        n = s["counts"].long()
        seq = torch.repeat_interleave(torch.arange(s["batch"], device=DEV), n, output_size=s["q"].shape[0])
        start = (n.cumsum(0) - n)[seq]
        pos = (s["lengths"].long() - n)[seq] + torch.arange(s["q"].shape[0], device=DEV) - start
        return _plain_rows(s, s["pages"][seq], pos)
    if s["op"] == "prefill":
        return _plain_prefill(s)
    if s["op"] == "pages":
        src, dst = (torch.tensor(s[x], device=DEV) for x in ("src", "dst"))
        pages = s["all"].view(s["caches"], s["pages"], -1)
        pages[:, dst] = pages[:, src]
        return s["all"]
    return _plain_logprobs(s)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    from accel_b200 import tensor as T
    if s["op"] == "pages":
        T.copy_pages(s["list"], s["src"], s["dst"], s["block"])
        return s["all"]
    if s["op"] == "logprobs":
        r = T.token_logprobs(s["x"], s["t"], top=s["top"])
        out = {"logprobs": r.logprobs, "entropy": r.entropy}
        if s["top"]:
            out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
        return out
    o = T.AttentionOptions(lengths=s["lengths"], pages=s.get("pages"), block=s["block"] if "pages" in s else 0,
                           scale=s["scale"], window=s["window"], sinks=s["sinks"])
    q = s["q"]
    if s["op"] == "decode":
        q = q[:, None]
    elif s["op"] == "ragged":
        o.query_extents = s["counts"]
    else:
        o.base = s["base"]
    return T.attention(q, s["k"], s["v"], o)


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "pages":
        out = s["all"].clone()
        for a, b in zip(s["src"], s["dst"]):
            out[:, b * c["block"]:(b + 1) * c["block"]] = s["all"][:, a * c["block"]:(a + 1) * c["block"]]
        return out
    if c["op"] == "logprobs":
        parts = [[], [], [], []]
        step = max(1, (1 << 24) // c["vocab"])
        for r in range(0, c["rows"], step):
            x = s["x"][r:r + step].double()
            lse = torch.logsumexp(x, 1)
            prob = torch.exp(x - lse[:, None])
            parts[0].append(x.gather(1, s["t"].view(c["rows"], -1)[r:r + step].long()) - lse[:, None])
            parts[1].append(lse - torch.where(prob > 0, prob * x, 0.0).sum(1))
            best = torch.argsort(x, dim=1, descending=True, stable=True)[:, :c["top"]]
            parts[2].append(best.int())
            parts[3].append(x.gather(1, best) - lse[:, None])
        lp, h, ids, top = (torch.cat(p) for p in parts)
        out = {"logprobs": lp.view(s["t"].shape), "entropy": h}
        if c["top"]:
            out["top_ids"], out["top_logprobs"] = ids, top
        return out
    rows, ln = _row_positions(c)
    blk, heads, group = c["block"], c["kv"] * c["group"], c["group"]
    paged = "pages" in s
    table = (s["pages"].view(len(ln), -1).long() if paged else None)
    out = torch.empty(len(rows), heads, c["dim"], dtype=torch.float64, device=DEV)
    by_seq = {}
    for r, (b, p) in enumerate(rows):
        by_seq.setdefault(b, []).append((r, p))
    for b, rp in by_seq.items():
        p0, p1 = rp[0][1], rp[-1][1]
        first = max(p0 - c["window"] + 1, 0)
        keys = list(range(min(c["sinks"], first))) + list(range(first, p1 + 1))
        j = torch.tensor(keys, device=DEV)
        where = table[b][j // blk] * blk + j % blk if paged else j
        p = torch.arange(p0, p1 + 1, device=DEV)[:, None]
        hidden = (j > p) | ((p - j >= c["window"]) & (j >= c["sinks"]))
        for h in range(heads):
            kh, vh = s["k"][where, h // group].double(), s["v"][where, h // group].double()
            for a in range(0, len(rp), 2048):
                m = rp[a:a + 2048]
                z = s["q"][m[0][0]:m[-1][0] + 1, h].double() @ kh.T * s["scale"]
                z[hidden[a:a + 2048]] = -math.inf
                out[m[0][0]:m[-1][0] + 1, h] = torch.softmax(z, 1) @ vh
    return out
