"""The operators that score, hold and share long contexts, and the work that is timed when their speed is looked at: the log probabilities of
given tokens with entropy and alternatives, a key/value cache held in 4 bits (written, read back, attended to), and the copying of cache
pages.  Each is here in its plain form -- elementary torch operations -- and as the call that a user makes of nano_b200.ops.

The cache in 4 bits, as both forms read it: a pool is bytes [pages][key/value heads][1280 n], n = head_dim / 32.  The block of one page and head is
    key codes [32 tokens][16 n] | key pairs [32 tokens][n] of two float16 | value codes [32 tokens][16 n] | value pairs [32 tokens][n]
and a group of 32 neighbouring coordinates x of one token and head is held as 4-bit codes c and the pair (s, m):
    m = f16(min x),  s = f16((max x - min x) * f32(1/15)),  c = min(15, max(0, round_half_even((x - m) / s))),  c = 0 where s = 0;   it stands for c s + m.
Coordinate 32 j + 8 b + i of a key is nibble i (from the lowest) of the little-endian 32-bit word b n + j of its codes; coordinate 32 j + 4 b + i of a
value is nibble i of the 16-bit word b n + j."""
import math

import torch

own = False

PAGE, GROUP = 32, 32


def listed():
    return [
        # a step of a served request: one row of logits over the largest vocabulary that this repository serves, five alternatives
        dict(name="logprobs one row", op="logprobs", rows=1, vocab=151936, type="f32", top=5, masked=0.0),
        # a batch of wanted places as the engine's classifier leaves them, the tokens' log probabilities alone
        dict(name="logprobs 64 rows", op="logprobs", rows=64, vocab=32000, type="f32", top=0, masked=0.0),
        # constrained decoding: most of an odd vocabulary is masked, in some rows all of it
        dict(name="logprobs masked odd", op="logprobs", rows=77, vocab=50257, type="bf16", top=8, masked=0.97),
        # a document is scored: every position with its twenty alternatives
        dict(name="logprobs document", op="logprobs", rows=1024, vocab=151936, type="bf16", top=20, masked=0.0),
        # the new tokens of 16 requests go to the cache, and come back as what they stand for
        dict(name="kv4 write 16 tokens", op="write", tokens=16, kv_heads=8, dim=128, type="bf16", skip=0.0),
        # a long portion of prompts, some of its rows padding
        dict(name="kv4 write prompt", op="write", tokens=9001, kv_heads=8, dim=128, type="f32", skip=0.1),
        # the next token of one chat
        dict(name="kv4 decode chat", op="attention", batch=1, tokens=1, heads=16, kv_heads=8, dim=128, context=777, window=0, softcap=0.0, sinks=False, ragged=False),
        # the next tokens of 32 requests of all lengths
        dict(name="kv4 decode batch", op="attention", batch=32, tokens=1, heads=32, kv_heads=8, dim=128, context=8190, window=0, softcap=0.0, sinks=False, ragged=True),
        # one request far into a very long context
        dict(name="kv4 decode long", op="attention", batch=1, tokens=1, heads=32, kv_heads=8, dim=128, context=131000, window=0, softcap=0.0, sinks=False, ragged=False),
        # a portion of a prompt behind what came before it, in layers with a window, capped scores and sinks
        dict(name="kv4 prompt portion", op="attention", batch=1, tokens=1000, heads=16, kv_heads=4, dim=64, context=4100, window=2500, softcap=30.0, sinks=True, ragged=False),
        # a prompt is forked for seven continuations: their last pages in every layer
        dict(name="pages fork", op="pages", pairs=7, pools=28, page_bytes=40960),
        # many pages move at once
        dict(name="pages many", op="pages", pairs=1000, pools=8, page_bytes=40960),
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    op = rng.choice(["logprobs", "logprobs", "write", "attention", "attention", "attention", "pages"])
    if op == "logprobs":
        vocab = rng.choice([spread(100, 151936), 32000, 151936])
        return dict(op=op, rows=spread(1, max(1, min(2048, 150_000_000 // vocab))), vocab=vocab, type=rng.choice(["f32", "bf16"]), top=rng.choice([0, rng.randint(1, 32)]),
                    masked=rng.choice([0.0, 0.0, rng.uniform(0.1, 0.99)]))
    if op == "write":
        return dict(op=op, tokens=spread(1, 9000), kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([32, 64, 96, 128]), type=rng.choice(["bf16", "f32"]), skip=rng.choice([0.0, rng.uniform(0.0, 0.5)]))
    if op == "pages":
        return dict(op=op, pairs=spread(1, 1000), pools=rng.randint(1, 8), page_bytes=16 * spread(4, 2560))
    kv_heads, rep = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 8])
    case = dict(op=op, heads=kv_heads * rep, kv_heads=kv_heads, dim=rng.choice([32, 64, 64, 96, 128, 128, 128, 256]), window=rng.choice([0, 0, spread(1, 4000)]),
                softcap=rng.choice([0.0, 0.0, 30.0]), sinks=rng.random() < 0.3, ragged=rng.random() < 0.5)
    if rng.random() < 0.6:          # single tokens
        case.update(batch=spread(1, 48), tokens=1)
        case["context"] = spread(1, max(2, min(100_000, 100_000_000 // (case["batch"] * kv_heads * case["dim"]))))
    else:
        case.update(batch=rng.randint(1, 3), tokens=spread(2, 700))
        case["context"] = case["tokens"] + spread(1, 2000)
    return case


# ---- inputs ----
def _type(case):
    return {"f32": torch.float32, "bf16": torch.bfloat16}[case["type"]]


def _quantise(x):
    """Rows of coordinates [..., dim] as codes [..., dim] and the pairs' halves [..., dim / 32] (float16)."""
    x = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = x.amin(-1), x.amax(-1)
    m, s = lo.half(), ((hi - lo) * (1.0 / 15.0)).half()
    step = torch.where(s > 0, s, torch.ones_like(s)).double()[..., None]
    c = ((x.double() - m.double()[..., None]) / step).round().clamp(0, 15) * (s > 0)[..., None]
    return c.flatten(-2).to(torch.uint8), s, m


def _nibbles(c, per):
    """Codes [..., dim] as bytes [..., dim / 2], `per` neighbouring coordinates to a word."""
    dim = c.shape[-1]
    w = c.unflatten(-1, (dim // GROUP, GROUP // per, per)).transpose(-3, -2).reshape(*c.shape[:-1], dim // 2, 2)
    return w[..., 0] | w[..., 1] << 4


def _blocks(k, v):
    """Keys and values [pages, 32, heads, dim] as a pool [pages, heads, 1280 dim / 32]."""
    def part(x, per):
        c, s, m = _quantise(x.transpose(1, 2))
        return _nibbles(c, per).flatten(2), torch.stack([s, m], -1).view(torch.uint8).flatten(2)
    return torch.cat([*part(k, 8), *part(v, 4)], -1)


def _values(pool, dim):
    """What a pool's blocks [pages, heads, bytes] stand for: keys and values [pages, 32, heads, dim] in 32 bits."""
    n = dim // GROUP

    def part(at, per):
        w = pool[..., at:at + PAGE * 16 * n].unflatten(-1, (PAGE, 16 * n))
        c = torch.stack([w & 15, w >> 4], -1).flatten(-2).unflatten(-1, (GROUP // per, n, per)).transpose(-3, -2).float()          # [pages, heads, 32, n, per words, per]
        sm = pool[..., at + PAGE * 16 * n:at + PAGE * 20 * n].contiguous().view(torch.float16).float().unflatten(-1, (PAGE, n, 2))
        return (c * sm[..., 0, None, None] + sm[..., 1, None, None]).flatten(-3).transpose(1, 2)
    return part(0, 8), part(PAGE * 20 * n, 4)


def _pool(gen, pages, heads, dim):
    """Pages as decoding leaves them: normal coordinates, channels with means of their own."""
    def rows():
        mean = torch.randn(1, 1, heads, dim, device="cuda", generator=gen) * 0.5
        return torch.randn(pages, PAGE, heads, dim, device="cuda", generator=gen) + mean
    return _blocks(rows(), rows())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case=case)
    if case["op"] == "logprobs":
        R, V = case["rows"], case["vocab"]
        x = torch.randn(R, V, device="cuda", generator=gen) * 2.5
        x.scatter_add_(1, torch.randint(0, V, (R, 8), device="cuda", generator=gen), torch.rand(R, 8, device="cuda", generator=gen) * 12)          # a few likely tokens
        if case["masked"]:
            x.masked_fill_(torch.rand(R, V, device="cuda", generator=gen) < case["masked"], -math.inf)
            x[5::31] = -math.inf
        st["logits"] = x.to(_type(case))
        st["tokens"] = torch.randint(0, V, (R,), device="cuda", generator=gen)
    elif case["op"] == "write":
        T, G, D = case["tokens"], case["kv_heads"], case["dim"]
        pages = (T + PAGE - 1) // PAGE + 3
        for name in ("k", "v"):
            st[name] = (torch.randn(T, G, D, device="cuda", generator=gen) + torch.randn(1, G, D, device="cuda", generator=gen)).to(_type(case))
        order = torch.randperm(pages, device="cuda", generator=gen)
        t = torch.arange(T, device="cuda")
        slots = order[t // PAGE] * PAGE + t % PAGE
        skipped = torch.rand(T, device="cuda", generator=gen) < case["skip"]
        st["slots"] = torch.where(skipped, torch.full_like(slots, -1), slots).int()          # places without a row are padding
        st["pool"] = torch.zeros(pages, G, 1280 * (D // GROUP), dtype=torch.uint8, device="cuda")
    elif case["op"] == "attention":
        B, T, H, G, D, n = case["batch"], case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["context"]
        width = (n + PAGE - 1) // PAGE
        lens = torch.full((B,), n, device="cuda")
        if case["ragged"]:          # every length up to the longest
            lens = torch.maximum((torch.rand(B, device="cuda", generator=gen) * n).long() + 1, torch.tensor(min(n, T), device="cuda"))
        pages = B * width + 2
        st["pool"] = _pool(gen, pages, G, D)
        st["table"] = torch.randperm(pages, device="cuda", generator=gen)[:B * width].view(B, width).int()
        st["lens"] = lens.int()
        st["q"] = (torch.randn(B, T, H, D, device="cuda", generator=gen) * 1.3).bfloat16()
        st["sinks"] = torch.randn(H, device="cuda", generator=gen) if case["sinks"] else None
    else:
        P, L, n = case["pairs"], case["pools"], case["page_bytes"]
        st["pools"] = torch.randint(0, 256, (L, 2 * P + 3, n), dtype=torch.uint8, device="cuda", generator=gen)
        order = torch.randperm(2 * P + 3, device="cuda", generator=gen)
        st["src_dev"], st["dst_dev"] = order[:P], order[P:2 * P]
        st["src"], st["dst"] = order[:P].tolist(), order[P:2 * P].tolist()          # the state manager's lists are on the host
    return st


# ---- the plain forms ----
def _logprobs(logits, tokens, top):
    x = logits.float()
    peak = x.amax(1, keepdim=True)
    empty = peak == -math.inf
    d = x - torch.where(empty, torch.zeros_like(peak), peak)
    e = d.exp()
    total = e.sum(1, keepdim=True)
    log_total = torch.where(empty, torch.zeros_like(total), total.log())
    lp = d.gather(1, tokens[:, None])[:, 0] - log_total[:, 0]
    spread = torch.where(e > 0, e * -d, torch.zeros_like(d)).sum(1)
    entropy = torch.where(empty[:, 0], torch.zeros_like(lp), log_total[:, 0] + spread / total[:, 0])
    best, ids = x.sort(dim=1, descending=True, stable=True) if top else (x[:, :0], tokens[:, None][:, :0])
    return lp, entropy, best[:, :top] - torch.where(empty, torch.zeros_like(peak), peak) - log_total, ids[:, :top].int()


def _attention(q, pool, table, lens, scale, window, softcap, sinks):
    B, T, H, D = q.shape
    G = pool.shape[1]
    k, v = _values(pool[table.long().flatten()], D)          # [B pages, 32, G, D]
    k, v = (x.reshape(B, -1, G, D).transpose(1, 2) for x in (k, v))
    qq = q.float().view(B, T, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, -1, D)          # rows: head of the group, then token
    s = (qq @ k.transpose(2, 3)).view(B, G, H // G, T, -1) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    at = torch.arange(s.shape[-1], device=q.device)
    pos = lens[:, None].long() - T + torch.arange(T, device=q.device)
    seen = at <= pos[:, :, None]
    if window:
        seen &= at > pos[:, :, None] - window
    s = torch.where(seen[:, None, None], s, torch.full_like(s, -math.inf))
    peak = s.amax(-1, keepdim=True)
    if sinks is not None:
        sink = sinks.view(1, G, H // G, 1, 1)
        peak = torch.maximum(peak, sink)
    e = (s - torch.where(peak == -math.inf, torch.zeros_like(peak), peak)).exp()
    total = e.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + (sink - peak).exp()
    p = torch.where(total > 0, e / total, torch.zeros_like(e))
    o = p.reshape(B, G, -1, p.shape[-1]) @ v
    return o.view(B, G, H // G, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(q.dtype)


def _written(k, v, slots, pool):
    """The pool's rows after the write, and what the written rows stand for (zeros where there is none)."""
    live = (slots >= 0)[:, None, None]

    def stands(x):
        c, s, m = _quantise(x)
        return torch.where(live, (c.float().unflatten(-1, (-1, GROUP)) * s.float()[..., None] + m.float()[..., None]).flatten(-2), torch.zeros((), device=x.device))
    n = k.shape[-1] // GROUP
    page, at, some = slots.clamp(min=0).long() // PAGE, slots.clamp(min=0).long() % PAGE, slots >= 0

    def put(x, off, per):
        c, s, m = _quantise(x)
        codes = pool[..., off:off + PAGE * 16 * n].unflatten(-1, (PAGE, 16 * n))
        pairs = pool[..., off + PAGE * 16 * n:off + PAGE * 20 * n].unflatten(-1, (PAGE, 4 * n))
        codes[page[some], :, at[some]] = _nibbles(c, per)[some]
        pairs[page[some], :, at[some]] = torch.stack([s, m], -1).view(torch.uint8).flatten(-2)[some]
    put(k, 0, 8)
    put(v, PAGE * 20 * n, 4)
    return stands(k), stands(v)


def run(st):
    c = st["case"]
    if own:
        from nano_b200 import ops
    if c["op"] == "logprobs":
        if own:
            return ops.token_logprobs(st["logits"], st["tokens"], top=c["top"])
        return _logprobs(st["logits"], st["tokens"], c["top"])
    if c["op"] == "write":
        if own:
            ops.kv4_write(st["pool"], st["k"], st["v"], st["slots"])
            return ops.kv4_read(st["pool"], st["slots"])
        return _written(st["k"], st["v"], st["slots"], st["pool"])
    if c["op"] == "attention":
        scale = c["dim"] ** -0.5
        if own:
            return ops.kv4_attention(st["q"], st["pool"], st["table"], st["lens"], scale=scale, window=c["window"], softcap=c["softcap"], sinks=st["sinks"])
        return _attention(st["q"], st["pool"], st["table"], st["lens"], scale, c["window"], c["softcap"], st["sinks"])
    if own:
        ops.pages_copy(list(st["pools"]), st["src"], st["dst"])
    else:
        st["pools"][:, st["dst_dev"]] = st["pools"][:, st["src_dev"]]
    return st["pools"]


def work(case):
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["type"] == "f32" else 2) + case["rows"] * (16 + 8 * case["top"]), "flops": 6 * n}
    if case["op"] == "write":
        n = case["tokens"] * case["kv_heads"] * case["dim"] * 2
        return {"bytes": n * (4 if case["type"] == "f32" else 2) + 2 * n * 5 // 8 + 4 * n, "flops": 6 * n}
    if case["op"] == "attention":
        B, T, H, G, D, n = case["batch"], case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["context"]
        mean = n * 0.5 if case["ragged"] else n          # lengths are spread evenly
        keys = sum(min(case["window"] or n, max(1.0, mean - t)) for t in range(T)) if T > 1 else min(case["window"] or n, mean)
        held = min(mean, (case["window"] or n) + T)
        return {"bytes": B * held * G * D * 2 * 5 / 8 + 2 * B * T * H * D * 2, "flops": B * 4 * keys * H * D}
    return {"bytes": 2 * case["pairs"] * case["pools"] * case["page_bytes"], "flops": 0}


# ---- the definitions in 64 bits ----
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "logprobs":
        lps, ents, tops = [], [], []
        for row, token in zip(st["logits"], st["tokens"].tolist()):
            x = row.double()
            z = torch.logsumexp(x, 0)
            x = x - z if z > -math.inf else x
            p = x.exp()
            lps.append(x[token])
            ents.append(-(p * torch.where(p > 0, x, torch.zeros_like(x))).sum())
            tops.append(torch.topk(x, case["top"]).values)
        return torch.stack(lps), torch.stack(ents), torch.stack(tops), None
    if case["op"] == "write":
        def stands(x):
            g = x.double().view(-1, GROUP)
            lo, hi = g.min(1, keepdim=True).values, g.max(1, keepdim=True).values
            s, m = (((hi - lo).float() * torch.tensor(1 / 15, device="cuda")).half().double(), lo.float().half().double())
            best, value = torch.full_like(g, math.inf), m + 0 * g
            for c in range(16):          # the nearest of the sixteen; of two as near the even one
                far = (g - (c * s + m)).abs()
                take = (s > 0) & ((far < best) | ((far == best) & (c % 2 == 0)))
                best, value = torch.where(take, far, best), torch.where(take, c * s + m, value)
            return value.view(x.shape) * (st["slots"] >= 0)[:, None, None]
        return stands(st["k"]), stands(st["v"])
    if case["op"] == "attention":
        B, T, H, G, D = (case[i] for i in ("batch", "tokens", "heads", "kv_heads", "dim"))
        n, pool = D // GROUP, st["pool"]
        d = torch.arange(D, device="cuda")
        token = torch.arange(PAGE, device="cuda")[:, None]
        out = torch.zeros(B, T, H, D, dtype=torch.float64, device="cuda")

        def row(block, at, per):          # [pages, bytes] -> [32 pages, D]
            nib = per * ((d % 32) // per * n + d // 32) + d % per
            byte = block[:, at + token * 16 * n + nib // 2].long()
            code = (byte >> (4 * (nib % 2))) & 15
            half = block[:, at + 512 * n:at + 640 * n].contiguous().view(torch.float16).double()
            return (code * half[:, (token * n + d // 32) * 2] + half[:, (token * n + d // 32) * 2 + 1]).reshape(-1, D)
        for b in range(B):
            keys = int(st["lens"][b])
            mine = pool[st["table"][b, :(keys + PAGE - 1) // PAGE].long()]
            pos = keys - T + torch.arange(T, device="cuda")[:, None]
            j = torch.arange(keys, device="cuda")[None]
            hidden = (j > pos) | (j <= pos - case["window"]) if case["window"] else j > pos
            for g in range(G):
                k, v = row(mine[:, g], 0, 8)[:keys], row(mine[:, g], 640 * n, 4)[:keys]
                for h in range(g * (H // G), (g + 1) * (H // G)):
                    s = st["q"][b, :, h].double() @ k.T * (float(D) ** -0.5)
                    if case["softcap"]:
                        s = case["softcap"] * torch.tanh(s / case["softcap"])
                    s = s.masked_fill(hidden, -math.inf)
                    if case["sinks"]:          # one more score that has no value
                        s = torch.cat([s, st["sinks"][h].double().expand(T, 1)], 1)
                    out[b, :, h] = torch.softmax(s, 1)[:, :keys].nan_to_num(0.0) @ v
        return out
    return None
