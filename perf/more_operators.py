"""The operators of products in microscaled 4-bit floating point and of routed experts, and the work that is timed when their speed is looked at: the quantisation, the
product of tokens with a matrix, tokens sorted by expert and back with their gradients, and the product of sorted tokens with the experts' matrices.  Each is here in its
plain form -- elementary torch operations -- and as the call that a user makes of nano_b200.ops.

The format, as both forms read it: a row's numbers are held in groups of 32 neighbours, the last one filled up with zeros.  A group has one byte E, which stands for the
scale 2^(E - 127) (255: NaN), and 32 codes of four bits, two to a byte, the lower four first: a sign and the number 0, 0.5, 1, 1.5, 2, 3, 4 or 6.  Of a group's largest
magnitude a the scale is 2^(floor(log2 a) - 2), between 2^-127 and 2^127 (2^-127 where a = 0); a code is the nearest to x / scale, of two as near the one with an even number, and
what lies beyond 6 becomes 6.  A group with a NaN or an infinity is NaN."""
import math

import torch

own = False

GROUP = 32
NUMBERS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # the state of one token, between two products of its layer
        dict(name="quantise one row", op="quantise", rows=1, columns=2560, type="bf16"),
        # a long prompt's activations in 32 bits, of an odd width: the last group is short
        dict(name="quantise prompt", op="quantise", rows=8191, columns=2570, type="f32"),
        # the next token of one request through a wide layer
        dict(name="product one token", op="product", rows=1, columns=2560, outputs=9728, type="bf16", out="bf16"),
        # the next tokens of 24 requests, their logits over the largest vocabulary that this repository serves
        dict(name="product batch", op="product", rows=24, columns=1024, outputs=151936, type="bf16", out="f32"),
        # a portion of a prompt, odd in every way, already in the format
        dict(name="product odd", op="product", rows=333, columns=1000, outputs=777, type="mx4", out="f32"),
        # a long prompt
        dict(name="product prompt", op="product", rows=8192, columns=2560, outputs=9728, type="bf16", out="bf16"),
        # the tokens of a decoding batch go to their experts
        dict(name="dispatch batch", op="dispatch", tokens=33, top=2, experts=16, columns=1024, type="bf16", dropped=0.0, grad=False),
        # a prompt's tokens, for a step that learns too: forward and backward
        dict(name="dispatch prompt", op="dispatch", tokens=8192, top=4, experts=64, columns=2048, type="bf16", dropped=0.02, grad=True),
        # what the experts said goes back to the tokens of a batch
        dict(name="combine batch", op="combine", tokens=33, top=2, experts=16, columns=1024, type="bf16", dropped=0.0, grad=False),
        # and to those of a prompt, forward and backward
        dict(name="combine prompt", op="combine", tokens=8192, top=4, experts=64, columns=2048, type="bf16", dropped=0.02, grad=True),
        # the experts of one token
        dict(name="experts one token", op="experts", tokens=1, top=4, experts=64, columns=2048, outputs=1024, type="bf16", out="bf16", dropped=0.0),
        # the experts of a prompt's tokens, some asked for much more than others
        dict(name="experts prompt", op="experts", tokens=4096, top=4, experts=64, columns=2048, outputs=1024, type="bf16", out="bf16", dropped=0.02),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantise", "product", "product", "product", "dispatch", "combine", "experts", "experts"])
    if op == "quantise":
        columns = _spread(rng, 1, 9728)
        return dict(op=op, rows=_spread(rng, 1, max(1, min(8192, 20_000_000 // columns))), columns=columns, type=rng.choice(["bf16", "f16", "f32"]))
    if op == "product":
        columns = rng.choice([_spread(rng, 32, 9728), 32 * _spread(rng, 1, 304)])
        outputs = _spread(rng, 16, max(16, min(151936, 150_000_000 // columns)))
        rows = _spread(rng, 1, max(1, min(8192, 200_000_000_000 // (columns * outputs), 60_000_000 // outputs)))
        return dict(op=op, rows=rows, columns=columns, outputs=outputs, type=rng.choice(["bf16", "bf16", "f32", "mx4"]), out=rng.choice(["bf16", "f32"]))
    top, experts = rng.choice([1, 2, 4, 8]), rng.choice([8, 16, 64, 128, rng.randint(8, 200)])
    case = dict(op=op, top=top, experts=experts, dropped=rng.choice([0.0, rng.uniform(0.0, 0.3)]))
    if op == "experts":
        columns, outputs = 8 * _spread(rng, 4, 256), _spread(rng, 16, 2048)
        while experts * columns * outputs > 134_000_000:
            columns, outputs = max(32, columns // 2), max(16, outputs // 2)
        rows = _spread(rng, 1, max(1, min(16384 // top, 34_000_000_000 // (columns * outputs * top))))
        return dict(case, tokens=rows, columns=columns, outputs=outputs, type=rng.choice(["bf16", "mx4"]), out=rng.choice(["bf16", "f32"]))
    columns = _spread(rng, 16, 4096)
    return dict(case, tokens=_spread(rng, 1, max(1, min(16384, 60_000_000 // (columns * top)))), columns=columns, type=rng.choice(["bf16", "f32"]), grad=rng.random() < 0.5)


# ---- inputs ----
def _type(name):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _groups(x):
    """Rows in 32 bits as [..., groups, 32], the last group filled up with zeros."""
    x = x.float()
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % GROUP)).unflatten(-1, (-1, GROUP))


def _power(e):
    """2^e in 32 bits, -127 <= e <= 127."""
    return torch.where(e < -126, torch.full_like(e, 1 << 22), (e + 127) << 23).int().view(torch.float32)


def _quantise(x):
    """The numbers of the codes (signed, [..., groups, 32]) and the exponents of the scales (whole numbers, [..., groups])."""
    x = _groups(x)
    top = x.abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, torch.full_like(top, -127).int()).clamp(-127, 127)          # frexp: top = m 2^exponent, 0.5 <= m < 1
    half = -e // 2
    a = x.abs() * _power(half)[..., None] * _power(-e - half)[..., None]          # (in two steps: 2^-e may lie beyond the type)
    n = torch.where(a < 2, (a * 2).round() * 0.5, torch.where(a < 4, a.round(), (a * 0.5).round() * 2)).clamp(max=6)          # (ties to even)
    bad = ~torch.isfinite(top)
    return torch.where(bad[..., None], torch.full_like(n, math.nan), n * torch.where(x < 0, -1.0, 1.0)), torch.where(bad, torch.full_like(e, 128), e)


def _stand_for(x):
    """What rows become in the format, in 32 bits."""
    n, e = _quantise(x)
    return (n * _power(e.clamp(max=127))[..., None]).flatten(-2)[..., :x.shape[-1]]


def _bytes(x):
    """Rows as codes and scales in bytes."""
    n, e = _quantise(x)
    a = n.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a * 0.5 + 4)).nan_to_num(0.0).to(torch.uint8) | (n < 0).to(torch.uint8) << 3
    code = code.flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, (e + 127).to(torch.uint8)


def _values(codes, scales, columns):
    """What codes and scales stand for, in 32 bits."""
    table = torch.tensor(NUMBERS + tuple(-v for v in NUMBERS), device=codes.device)
    v = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()
    s = torch.where(scales == 255, torch.full(scales.shape, math.nan, device=codes.device), _power((scales.int() - 127).clamp(max=127)))
    return (table[v].unflatten(-1, (-1, GROUP)) * s[..., None]).flatten(-2)[..., :columns]


def _rows(gen, rows, columns):
    """Activations: normal numbers, channels of different size, a few outliers."""
    x = torch.randn(rows, columns, device="cuda", generator=gen) * (torch.randn(columns, device="cuda", generator=gen) * 0.7).exp()
    return torch.where(torch.rand(rows, columns, device="cuda", generator=gen) < 1e-3, x * 20, x)


def _routing(gen, case):
    """Experts of each token, without repetition, some much more asked for; -1 where a token has fewer."""
    T, k, E = case["tokens"], case["top"], case["experts"]
    liking = torch.randn(E, device="cuda", generator=gen) * 0.7
    noise = -torch.log(-torch.log(torch.rand(T, E, device="cuda", generator=gen).clamp(1e-9, 1 - 1e-7)))
    ids = (liking + noise).topk(k, 1).indices
    return torch.where(torch.rand(T, k, device="cuda", generator=gen) < case["dropped"], torch.full_like(ids, -1), ids)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st, op = dict(case=case), case["op"]
    if op == "quantise":
        st["x"] = _rows(gen, case["rows"], case["columns"]).to(_type(case["type"]))
        return st
    if op == "product":
        w = torch.randn(case["outputs"], case["columns"], device="cuda", generator=gen) * case["columns"] ** -0.5
        st["codes"], st["scales"] = _bytes(w)          # laid out once, as a program holds its weights
        x = _rows(gen, case["rows"], case["columns"])
    else:
        st["ids"] = _routing(gen, case)
        st["order"], st["offsets"], st["place"] = _sorted(st["ids"], case["experts"])
        R = st["order"].shape[0]
        if op == "experts":
            st["most"] = int((st["offsets"][1:] - st["offsets"][:-1]).max())
            w = torch.randn(case["experts"], case["outputs"], case["columns"], device="cuda", generator=gen) * case["columns"] ** -0.5
            st["codes"], st["scales"] = _bytes(w)
            x = _rows(gen, R, case["columns"])
        else:
            kind = _type(case["type"])
            st["x"] = torch.randn(case["tokens"] if op == "dispatch" else R, case["columns"], device="cuda", generator=gen).to(kind)
            st["weights"] = torch.softmax(torch.randn(case["tokens"], case["top"], device="cuda", generator=gen), 1)
            if case["grad"]:
                st["x"].requires_grad_()
                st["weights"].requires_grad_()
                st["g"] = torch.randn(R if op == "dispatch" else case["tokens"], case["columns"], device="cuda", generator=gen).to(kind)
            return st
    del w
    if case["type"] == "mx4":
        st["x"] = _bytes(x)
    else:
        st["x"] = x.to(_type(case["type"]))
    return st


# ---- the plain forms ----
def _sorted(ids, experts):
    flat = ids.flatten().long()
    n = flat.numel()
    known = (flat >= 0) & (flat < experts)
    key = torch.where(known, flat, torch.full_like(flat, experts))
    by, order = key.sort(stable=True)
    offsets = torch.searchsorted(by, torch.arange(experts + 1, device=ids.device)).int()
    place = torch.empty_like(order).scatter_(0, order, torch.arange(n, device=ids.device))
    return torch.where(by < experts, order, torch.full_like(order, -1)).int(), offsets, torch.where(known, place, torch.full_like(place, -1)).int().view_as(ids)


def _gathered(x, order, top):
    """Rows order[r] / top of x in 32 bits, zeros where there is none."""
    return torch.where((order >= 0)[:, None], x[order.clamp(min=0).long() // top].float(), torch.zeros((), device=x.device))


def _at_places(y, place):
    """y's rows by token, [tokens, top, columns] in 32 bits, zeros where there is none."""
    return torch.where((place >= 0)[..., None], y[place.clamp(min=0).long()].float(), torch.zeros((), device=y.device))


def _plain_rows(x, case):
    """The tokens as what their codes stand for."""
    if case["type"] == "mx4":
        return _values(*x, case["columns"])
    return _stand_for(x)


def _experts(x, w, offsets, most):
    """Rows by expert, [experts, most, columns], times the experts' matrices, and back."""
    E, R = w.shape[0], x.shape[0]
    r = torch.arange(R, device=x.device)
    e = torch.searchsorted(offsets.long(), r, right=True) - 1
    live = e < E
    e = e.clamp(max=E - 1)
    at = torch.where(live, e * max(most, 1) + r - offsets[e], torch.zeros_like(r))
    padded = torch.zeros(E * max(most, 1) + 1, x.shape[1], device=x.device)
    padded[torch.where(live, at, torch.full_like(at, E * max(most, 1)))] = x
    y = torch.bmm(padded[:-1].view(E, -1, x.shape[1]), w.transpose(1, 2)).view(-1, w.shape[1])
    return torch.where(live[:, None], y[at], torch.zeros((), device=x.device))


def run(st):
    c = st["case"]
    if own:
        from nano_b200 import ops
    if c["op"] == "quantise":
        if own:
            return ops.mx4_read(ops.mx4_quantize(st["x"]))
        return _stand_for(st["x"])
    if c["op"] in ("product", "experts"):
        out = _type(c["out"])
        if own:
            x, w = ops.Mx4(*st["x"], c["columns"]) if c["type"] == "mx4" else st["x"], ops.Mx4(st["codes"], st["scales"], c["columns"])
            return ops.mx4_product(x, w, dtype=out) if c["op"] == "product" else ops.experts_product(x, w, st["offsets"], dtype=out)
        x, w = _plain_rows(st["x"], c), _values(st["codes"], st["scales"], c["columns"])
        return (x @ w.T if c["op"] == "product" else _experts(x, w, st["offsets"], st["most"])).to(out)
    if c["op"] == "dispatch":
        if own:
            routing = ops.experts_sort(st["ids"], c["experts"])
            xs = ops.experts_gather(st["x"], routing)
            grads = torch.autograd.grad(xs, [st["x"]], st["g"]) if c["grad"] else []
            return [*routing, xs.detach(), *grads]
        x = st["x"].detach()
        order, offsets, place = _sorted(st["ids"], c["experts"])
        grads = [_at_places(st["g"], place).sum(1).to(x.dtype)] if c["grad"] else []
        return [order, offsets, place, _gathered(x, order, c["top"]).to(x.dtype), *grads]
    if own:
        out = ops.experts_combine(st["x"], ops.Routing(st["order"], st["offsets"], st["place"]), st["weights"])
        return [out.detach(), *(torch.autograd.grad(out, [st["x"], st["weights"]], st["g"]) if c["grad"] else [])]
    y, weights = _at_places(st["x"].detach(), st["place"]), st["weights"].detach()
    out = [(y * weights[..., None]).sum(1).to(st["x"].dtype)]
    if c["grad"]:
        g = st["g"].float()
        w = torch.where(st["order"] >= 0, weights.flatten()[st["order"].clamp(min=0).long()], torch.zeros((), device=g.device))
        out += [(_gathered(g, st["order"], c["top"]) * w[:, None]).to(st["x"].dtype), (y * g[:, None]).sum(2)]
    return out


def work(case):
    size = {"f32": 4.0, "bf16": 2.0, "f16": 2.0, "mx4": 17 / 32}[case["type"]]
    K = case["columns"]
    if case["op"] == "quantise":
        n = case["rows"] * K
        return {"bytes": n * (size + 2 * 17 / 32 + 4), "flops": 5 * n}
    if case["op"] == "product":
        M, N = case["rows"], case["outputs"]
        return {"bytes": N * K * 17 / 32 + M * K * size + M * N * (4 if case["out"] == "f32" else 2), "flops": 2 * M * N * K}
    T, k, E = case["tokens"], case["top"], case["experts"]
    R = T * k
    if case["op"] == "experts":
        N, asked = case["outputs"], min(E, E * (1 - (1 - k / E) ** T))          # experts that some token asks for, were all asked for alike
        return {"bytes": asked * N * K * 17 / 32 + R * K * size + R * N * (4 if case["out"] == "f32" else 2), "flops": 2 * R * N * K}
    if case["op"] == "dispatch":
        return {"bytes": R * 16 + 4 * E + (1 + case["grad"]) * (T + R) * K * size, "flops": R * K * case["grad"]}
    return {"bytes": R * (8 + 8 * case["grad"]) + (T + R) * K * size + case["grad"] * (T + 2 * R) * K * size, "flops": (2 + 3 * case["grad"]) * R * K}


# ---- the definitions in 64 bits ----
def _nearest(x):
    """What numbers [..., columns] become in the format, in 64 bits: the nearest of the sixteen, of two as near the one with an even number."""
    K = x.shape[-1]
    G = -(-K // GROUP)
    g = torch.zeros(*x.shape[:-1], G * GROUP, dtype=torch.float64, device=x.device)
    g[..., :K] = x.double()
    g = g.view(*x.shape[:-1], G, GROUP)
    top = g.abs().max(-1, keepdim=True).values
    e = torch.clamp(torch.floor(torch.log2(top)), -200, 200)
    e = e + (torch.exp2(e + 1) <= top).double() - (torch.exp2(e) > top).double()          # (log2 may land beside a power of two)
    scale = torch.exp2(torch.clamp(e - 2, -127, 127))
    a, best, far = g.abs() / scale, torch.zeros_like(g), torch.full_like(g, math.inf)
    for i, v in enumerate(NUMBERS):
        d = (a - v).abs()
        take = (d < far) | ((d == far) & (i % 2 == 0))
        best, far = torch.where(take, torch.full_like(best, v), best), torch.where(take, d, far)
    return (torch.copysign(best, g) * scale).reshape(*x.shape[:-1], -1)[..., :K]


def _meaning(codes, scales, columns):
    b = codes.long()
    out = torch.zeros(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        n = (b >> (4 * half)) & 15
        e, m = (n >> 1) & 3, n & 1
        out[..., half::2] = torch.where(e > 0, (1 + 0.5 * m) * torch.exp2(e.double() - 1), 0.5 * m) * (1 - 2 * (n >> 3))
    return (out.view(*codes.shape[:-1], -1, GROUP) * torch.exp2(scales.double() - 127)[..., None]).reshape(out.shape)[..., :columns]


def exact(case, seed):
    st = prepare(case, seed)
    c, K = case, case["columns"]
    if c["op"] == "quantise":
        return _nearest(st["x"])
    if c["op"] in ("product", "experts"):
        def tokens(r0, r1):
            return _meaning(st["x"][0][r0:r1], st["x"][1][r0:r1], K) if c["type"] == "mx4" else _nearest(st["x"][r0:r1])
        if c["op"] == "product":
            y = torch.zeros(c["rows"], c["outputs"], dtype=torch.float64, device="cuda")
            x = tokens(0, c["rows"])
            for n in range(0, c["outputs"], 8192):
                y[:, n:n + 8192] = x @ _meaning(st["codes"][n:n + 8192], st["scales"][n:n + 8192], K).T
            return y
        y = torch.zeros(st["order"].shape[0], c["outputs"], dtype=torch.float64, device="cuda")
        at = st["offsets"].tolist()
        for e in range(c["experts"]):
            if at[e + 1] > at[e]:
                y[at[e]:at[e + 1]] = tokens(at[e], at[e + 1]) @ _meaning(st["codes"][e], st["scales"][e], K).T
        return y
    T, k = c["tokens"], c["top"]
    x, place, ids = st["x"].detach().double(), st["place"].cpu(), st["ids"].cpu()
    live = ((ids >= 0) & (ids < c["experts"])).cuda()
    where = torch.zeros(T, k, dtype=torch.long)          # places counted anew: by expert, and within one by token
    n = 0
    for e in range(c["experts"]):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        where[t, j] = n + torch.arange(t.numel())
        n += t.numel()
    where = where.cuda()
    if c["op"] == "dispatch":
        out = torch.zeros(T * k, K, dtype=torch.float64, device="cuda")
        back = torch.zeros(T, K, dtype=torch.float64, device="cuda")
        for j in range(k):
            on = live[:, j]
            out[where[on, j]] = x[on]
            if c["grad"]:
                back[on] += st["g"][where[on, j]].double()
        return [None, None, None, out] + ([back] if c["grad"] else [])
    w = st["weights"].detach().double()
    out, dy, dw = torch.zeros(T, K, dtype=torch.float64, device="cuda"), torch.zeros_like(x), torch.zeros_like(w)
    for j in range(k):
        on = live[:, j]
        rows = where[on, j]
        out[on] += w[on, j, None] * x[rows]
        if c["grad"]:
            dy[rows] = w[on, j, None] * st["g"][on].double()
            dw[on, j] = (x[rows] * st["g"][on].double()).sum(1)
    return [out] + ([dy, dw] if c["grad"] else [])
