"""Products in microscaled 4-bit floating point and routed experts (nano_b200.ops) against their definitions in 64 bits, at the sizes, strides, values and routings where they can go wrong.

Tolerances.  Quantisation is exact: its scales and numbers are fixed.  A product's terms are exact; adding K of them in 32 bits, in whatever order and cut off or rounded, is off by at most a step of
2^-23 of the sum of their magnitudes S at each addition: K 2^-23 S, and half a step of the result's type.  A token's sum over its `top` experts is off by top + 1 roundings of 2^-24 of its terms'
magnitudes, a scalar product over D columns by D + 1 of them, and each by half a step of its type."""
import math
import os
import subprocess
import sys

import pytest
import torch

from nano_b200 import ops
from nano_b200.engine import NB200Error

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
NUMBERS = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, kind="f32"):
    return torch.randn(*shape, device="cuda", generator=gen(seed)).to(DT[kind])


def near(got, want, tol, what):
    got, want = got.double(), want.double()
    ok = (got == want) | (got.isnan() & want.isnan()) | ((got - want).abs() <= tol)
    assert got.shape == want.shape
    assert ok.all(), f"{what}: {(~ok).sum()} of {ok.numel()} off, first at {torch.nonzero(~ok)[0].tolist()}: {got[~ok][:3].tolist()} for {want[~ok][:3].tolist()}"


def values(m):
    """What an Mx4 stands for, in 64 bits."""
    c, s = m.codes.cpu(), m.scales.cpu().double()
    v = NUMBERS[torch.stack([c & 15, c >> 4], -1).flatten(-2).long()]
    s = torch.where(s == 255, math.nan, torch.exp2(s - 127))
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)[..., :m.columns].cuda()


def quantised(x):
    """(scales' bytes, what x becomes in 64 bits)"""
    K = x.shape[-1]
    x = torch.nn.functional.pad(x.cpu().double(), (0, -K % 32)).unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    bad = ~top.isfinite()
    m, e = torch.frexp(torch.where(bad, 1.0, top))
    e = torch.where(top > 0, e - 3, -127).clamp(-127, 127)
    a = x.abs() / torch.exp2(e.double())[..., None]
    grid = NUMBERS[:8]
    d = (a[..., None] - grid).abs()
    best = d.amin(-1, keepdim=True)
    even = torch.arange(8) % 2 == 0
    pick = torch.where((d == best) & even, 0, torch.where(d == best, 1, 2)).argmin(-1)
    v = grid[pick] * torch.where(x < 0, -1.0, 1.0) * torch.exp2(e.double())[..., None]
    return torch.where(bad, 255, e + 127).to(torch.uint8).cuda(), torch.where(bad[..., None], math.nan, v).flatten(-2)[..., :K].cuda()


def random_mx4(*shape, seed=0, spread=8):
    """Codes of any kind, scales around 1."""
    K, G = shape[-1], -(-shape[-1] // 32)
    c = torch.randint(0, 256, (*shape[:-1], 16 * G), device="cuda", generator=gen(seed), dtype=torch.uint8)
    s = torch.randint(127 - spread, 128 + spread, (*shape[:-1], G), device="cuda", generator=gen(seed + 1), dtype=torch.uint8)
    if K % 32:          # what fills up the last group is zeros
        keep = torch.arange(32 * G, device="cuda") < K
        c = c & (keep[0::2] * 15 + keep[1::2] * 240).to(torch.uint8)
    return ops.Mx4(c, s, K)


# ---------------- quantisation ----------------
def check_quantised(x):
    m = ops.mx4_quantize(x)
    s, v = quantised(x)
    assert m.columns == x.shape[-1] and m.codes.shape == (*x.shape[:-1], 16 * s.shape[-1])
    assert torch.equal(m.scales, s)
    near(values(m), v, 0.0, "quantised")
    near(ops.mx4_read(m), v.float(), 0.0, "read")          # (fp32 holds every number of the format but those below 2^-149, of which there are none)
    return m


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,columns", [(1, 1), (3, 31), (2, 32), (5, 33), (257, 64), (1, 2560), (7, 1000), (300, 2570), (4097, 8)])
def test_quantise(kind, rows, columns):
    x = (torch.randn(rows, columns, device="cuda", generator=gen(rows)) * torch.randn(rows, 1, device="cuda", generator=gen(1)).exp()).to(DT[kind])
    check_quantised(x)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("offset,pad", [(1, 0), (3, 5), (0, 1), (7, 8), (2, 2), (4, 4)])
def test_quantise_rows_anywhere(kind, offset, pad):
    x = randn(37, 130 + offset + pad, seed=3, kind=kind)
    x[:, :offset] = math.nan          # what lies beside the rows is not looked at
    x[:, 130 + offset:] = math.nan
    check_quantised(x[:, offset:offset + 130])
    check_quantised(x.t().contiguous().t()[:, offset:offset + 130])
    check_quantised(x[:, offset:offset + 130].expand(2, 37, 130))
    check_quantised(x[0, offset:offset + 130])
    check_quantised(x[:1, offset:offset + 130].expand(9, 130))


def test_quantise_special_values():
    x = torch.zeros(24, 32, device="cuda")
    x[1, 3] = math.nan
    x[2, 5], x[3, 5] = math.inf, -math.inf
    x[4, :4] = torch.tensor([3.4e38, -3.4e38, 1e38, 1e37])
    x[5, :4] = torch.tensor([1e-45, -1e-45, 1e-39, 3e-39])          # below what the smallest scale resolves, and beside it
    x[6, :4] = torch.tensor([2.0 ** -126, 2.0 ** -127, 2.0 ** -128, -(2.0 ** -129)])
    x[7, :8] = torch.tensor([8.0, .25, .75, 1.25, 1.75, 2.5, 3.5, 5.0]) / 2 * 1.0          # halves between neighbours, at the scale of 4
    x[8, :9] = torch.tensor([7.9, .5, 1.5, 2.5, 3.5, 5.0, 7.0, -7.0, 6.5])
    x[9] = torch.linspace(-7.999, 7.999, 32)
    x[10] = torch.nextafter(torch.full((32,), 4.0), torch.tensor(0.0)).cuda()              # just below a power of two
    x[11] = 4.0
    x[12, 31] = -0.0
    x[13, 0], x[13, 1:] = 6.0, torch.tensor([0.25] * 15 + [0.25000003] * 16)
    x[14, 0], x[14, 1] = 1e30, 1e-30
    for i in range(9):
        x[15 + i] = torch.arange(32, device="cuda") * 0.125 * 2.0 ** (i * 25 - 110)
    check_quantised(x)
    check_quantised(x.bfloat16())
    check_quantised((x.clamp(-6e4, 6e4)).half())
    assert ops.mx4_quantize(x).scales[:4, 0].tolist() == [0, 255, 255, 255]


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("columns", [8192, 8190, 8188, 8191])
def test_read_everything(kind, columns):
    codes = torch.arange(256, device="cuda").to(torch.uint8).repeat(16).expand(256, 4096).contiguous()          # every byte, under every scale
    scales = torch.arange(256, device="cuda").to(torch.uint8)[:, None].expand(256, 256).contiguous()
    m = ops.Mx4(codes, scales, columns)
    got, want = ops.mx4_read(m, DT[kind]), values(m)
    assert got.dtype == DT[kind]
    near(got, want.float().to(DT[kind]), 0.0, "read")
    wide = ops.Mx4(torch.zeros(256, 4112, dtype=torch.uint8, device="cuda")[:, 16:], scales.repeat(1, 2)[:, 1:257], columns)
    wide.codes.copy_(codes)
    near(ops.mx4_read(wide, DT[kind]), want.float().to(DT[kind]), 0.0, "read of strided rows")


def test_quantise_nothing():
    for shape in [(0, 32), (3, 0), (0, 0), (2, 0, 64)]:
        m = ops.mx4_quantize(torch.zeros(shape, device="cuda"))
        assert ops.mx4_read(m).shape == shape


# ---------------- products ----------------
def check_product(x, w, dtype, offsets=None):
    xv = values(x) if isinstance(x, ops.Mx4) else quantised(x)[1]
    wv, K = values(w), w.columns
    got = ops.mx4_product(x, w, dtype) if offsets is None else ops.experts_product(x, w, offsets, dtype)
    if offsets is None:
        want, size = xv @ wv.T, xv.abs() @ wv.abs().T
    else:
        want = torch.zeros(xv.shape[0], wv.shape[1], dtype=torch.float64, device="cuda")
        size = torch.zeros_like(want)
        at = offsets.tolist()
        for e in range(wv.shape[0]):
            want[at[e]:at[e + 1]] = xv[at[e]:at[e + 1]] @ wv[e].T
            size[at[e]:at[e + 1]] = xv[at[e]:at[e + 1]].abs() @ wv[e].abs().T
    dtype = dtype or torch.bfloat16
    assert got.dtype == dtype
    fine = size.isfinite()
    near(got, want, torch.where(fine, K * 2.0 ** -23 * size + HALF[dtype] * want.abs() + 1e-44, 0.0), "product")
    again = ops.mx4_product(x, w, dtype) if offsets is None else ops.experts_product(x, w, offsets, dtype)
    assert torch.equal(got.view(torch.uint8), again.view(torch.uint8))          # no order of arrival in it
    return got


SIZES = [(1, 1, 1), (1, 128, 32), (2, 129, 33), (7, 127, 64), (16, 64, 31), (17, 300, 256), (24, 1000, 1024), (33, 16, 2560), (64, 128, 512), (65, 257, 255), (128, 256, 257), (129, 640, 96),
         (255, 130, 1000), (257, 1025, 320), (333, 777, 1000), (512, 512, 4096), (1000, 136, 288), (1, 9728, 2560), (3, 1536, 9728), (8, 5000, 640)]


@pytest.mark.parametrize("rows,outputs,columns", SIZES)
def test_product_of_codes(rows, outputs, columns):
    x, w = random_mx4(rows, columns, seed=rows), random_mx4(outputs, columns, seed=outputs + 7)
    check_product(x, w, torch.float32)
    check_product(x, w, torch.bfloat16)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,outputs,columns", [(1, 512, 1024), (5, 300, 1000), (40, 257, 352), (200, 384, 640)])
def test_product_of_numbers(kind, rows, outputs, columns):
    x, w = randn(rows, columns, seed=4, kind=kind), ops.mx4_quantize(randn(outputs, columns, seed=5))
    check_product(x, w, DT[kind])
    check_product(x, w, torch.float32)
    y = ops.mx4_product(x.view(rows, 1, columns).expand(rows, 2, columns), w)
    assert y.dtype == x.dtype and y.shape == (rows, 2, outputs) and torch.equal(y[:, 0], y[:, 1]) and torch.equal(y[:, 0], ops.mx4_product(x, w))
    assert torch.equal(ops.mx4_product(x[0], w), ops.mx4_product(x[:1], w)[0])


@pytest.mark.parametrize("rows", [1, 20, 150])
def test_product_of_rows_anywhere(rows):
    K, N = 480, 200
    big_x, big_w = random_mx4(rows, 1024, seed=1), random_mx4(2 * N, 1024, seed=2)
    x = ops.Mx4(big_x.codes[:, 16:16 + 240], big_x.scales[:, 5:20], K)
    w = ops.Mx4(big_w.codes[::2, 32:32 + 240], big_w.scales[::2, 7:22], K)
    check_product(x, w, torch.float32)
    t = ops.Mx4(x.codes, x.scales.t().contiguous().t()[:, :15].contiguous(), K)
    assert torch.equal(ops.mx4_product(t, w), ops.mx4_product(x, w))


@pytest.mark.parametrize("rows", [1, 20, 150])
def test_product_of_special_values(rows):
    K, N = 192, 140
    x, w = random_mx4(rows, K, seed=8), random_mx4(N, K, seed=9)
    w.scales[3, 2] = 255          # a group that is NaN makes its output NaN, and no other
    w.scales[7] = 0
    w.codes[9] = 0
    w.scales[9] = 254             # zeros at the largest scale
    w.scales[11] = 230
    x.scales[0, 1] = 20           # scales far apart
    got = check_product(x, w, torch.float32)
    assert got[:, 3].isnan().all() and not got[:, :3].isnan().any() and (got[:, 9] == 0).all()
    x.scales[rows - 1, 0] = 255
    got = check_product(x, w, torch.float32)
    assert got[rows - 1].isnan().all() and (rows == 1 or not got[:rows - 1, 4:].isnan().any())
    y = randn(rows, K, seed=3)
    y[rows // 2, 5] = math.inf
    assert check_product(y, w, torch.float32)[rows // 2].isnan().all()


def test_product_beside_memory_that_is_not_its_own():
    """Rows behind the last, groups behind the last and columns that fill up a group may hold anything: nothing of it shows."""
    for rows in (1, 19, 140):
        x, w = random_mx4(rows + 3, 256, seed=1), random_mx4(150, 256, seed=2)
        x.scales[rows:], w.scales[130:] = 255, 255
        x.scales[:, 5:], w.scales[:, 5:] = 255, 255
        a, b = ops.Mx4(x.codes[:rows, :80], x.scales[:rows, :5], 160), ops.Mx4(w.codes[:130, :80], w.scales[:130, :5], 160)
        check_product(a, b, torch.float32)


def test_product_of_nothing():
    w = random_mx4(40, 64)
    assert ops.mx4_product(torch.zeros(0, 64, device="cuda"), w).shape == (0, 40)
    assert ops.mx4_product(torch.zeros(3, 64, device="cuda"), ops.Mx4(w.codes[:0], w.scales[:0], 64)).shape == (3, 0)
    none = ops.mx4_quantize(torch.zeros(5, 0, device="cuda"))
    assert torch.equal(ops.mx4_product(torch.zeros(3, 0, device="cuda"), none), torch.zeros(3, 5, device="cuda"))


# ---------------- products of sorted rows ----------------
def offsets_of(counts, first=0):
    return torch.cat([torch.zeros(1, dtype=torch.long), torch.tensor(counts).cumsum(0)]).add(first).int().cuda()


@pytest.mark.parametrize("counts,tail", [([1], 0), ([0, 1, 0, 1], 0), ([0, 0, 0], 5), ([3, 0, 17, 1, 0, 129], 4), ([128, 128], 0), ([40] * 9, 1), ([0, 300, 0, 0, 1], 0), ([1] * 64, 0), ([2, 0] * 100, 3)])
@pytest.mark.parametrize("outputs,columns", [(16, 32), (200, 288), (257, 1000)])
def test_experts_product(counts, tail, outputs, columns):
    rows = sum(counts) + tail
    x, w = random_mx4(rows, columns, seed=rows), random_mx4(len(counts), outputs, columns, seed=3)
    got = check_product(x, w, torch.float32, offsets_of(counts))
    assert (got[rows - tail:] == 0).all()
    xf = randn(rows, columns, seed=5, kind="bf16")
    check_product(xf, w, torch.bfloat16, offsets_of(counts))


def test_experts_product_of_rows_anywhere():
    x, w = random_mx4(50, 1024, seed=1), random_mx4(6, 90, 1024, seed=2)
    part = ops.Mx4(w.codes[1::2, 5:75, 64:160], w.scales[1::2, 5:75, 3:9], 190)
    rows = ops.Mx4(x.codes[:, 16:112], x.scales[:, 2:8], 190)
    check_product(rows, part, torch.float32, offsets_of([7, 0, 33], first=4))          # (rows before the first are zeros too)
    assert (ops.experts_product(rows, part, offsets_of([7, 0, 33], first=4))[:4] == 0).all()


# ---------------- sorting, gathering, combining ----------------
def sorted_reference(ids, experts):
    flat = ids.flatten().cpu().long()
    known = (flat >= 0) & (flat < experts)
    key = torch.where(known, flat, experts)
    by, order = key.sort(stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(flat.numel())
    offsets = torch.bincount(key, minlength=experts + 1)[:experts].cumsum(0)
    return torch.where(by < experts, order, -1).int(), torch.cat([torch.zeros(1, dtype=torch.long), offsets]).int(), torch.where(known, place, -1).int().view(ids.shape)


@pytest.mark.parametrize("tokens,top,experts", [(0, 2, 4), (1, 1, 1), (1, 8, 128), (33, 2, 16), (31, 1, 3), (1000, 4, 64), (1024, 4, 1024), (4097, 1, 7), (2049, 2, 1000), (9000, 8, 256), (70000, 4, 200)])
@pytest.mark.parametrize("wide", [False, True])
def test_sort(tokens, top, experts, wide):
    ids = torch.randint(-2 if tokens % 2 else 0, experts + (tokens % 2), (tokens, top), device="cuda", generator=gen(tokens))
    ids = ids if wide else ids.int()
    for x in (ids, (ids % 3) * (experts - 1) // 2, torch.full_like(ids, experts - 1), torch.full_like(ids, -1)):
        got = ops.experts_sort(x, experts)
        for a, b in zip(got, sorted_reference(x, experts)):
            assert a.dtype == torch.int32 and torch.equal(a.cpu(), b)
    if wide and tokens:
        ids[0, 0] = 1 << 32          # no expert, though its lower half is one's number
        assert torch.equal(ops.experts_sort(ids, experts).place.cpu(), sorted_reference(ids, experts)[2])


def routing_of(tokens, top, experts, seed=0, dropped=0.2):
    ids = torch.randint(0, experts, (tokens, top), device="cuda", generator=gen(seed))
    ids[torch.rand(tokens, top, device="cuda", generator=gen(seed + 1)) < dropped] = -1
    return ids, ops.experts_sort(ids, experts)


def by_token(y, place):
    return torch.where((place >= 0)[..., None], y.double()[place.clamp(min=0).long()], 0.0)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tokens,top,columns", [(1, 1, 1), (1, 4, 2048), (33, 2, 1024), (100, 8, 267), (257, 3, 130), (70, 1, 36), (1000, 4, 520)])
@pytest.mark.parametrize("dropped", [0.0, 0.3, 1.0])
def test_gather_and_combine(kind, tokens, top, columns, dropped):
    _, r = routing_of(tokens, top, 9, seed=tokens, dropped=dropped)
    x = randn(tokens, columns, seed=1, kind=kind).requires_grad_()
    xs = ops.experts_gather(x, r)
    want = torch.where((r.order >= 0)[:, None], x.detach()[r.order.clamp(min=0).long() // top], torch.zeros((), device="cuda", dtype=x.dtype))
    assert torch.equal(xs.detach(), want) and torch.equal(ops.experts_gather(x.detach(), r), want)
    g = randn(tokens * top, columns, seed=2, kind=kind)
    dx, = torch.autograd.grad(xs, x, g)
    parts = by_token(g, r.place)
    near(dx, parts.sum(1), (top + 1) * 2.0 ** -24 * parts.abs().sum(1) + HALF[x.dtype] * parts.sum(1).abs() + 1e-44, "gradient of gather")

    y = randn(tokens * top, columns, seed=3, kind=kind).requires_grad_()
    w = randn(tokens, top, seed=4).requires_grad_()
    out = ops.experts_combine(y, r, w)
    parts = by_token(y.detach(), r.place) * w.detach().double()[..., None]
    near(out.detach(), parts.sum(1), (top + 1) * 2.0 ** -24 * parts.abs().sum(1) + HALF[x.dtype] * parts.sum(1).abs() + 1e-7 * (kind == "f16"), "combined")
    assert torch.equal(ops.experts_combine(y.detach(), r, w.detach()), out.detach())
    g = randn(tokens, columns, seed=5, kind=kind)
    dy, dw = torch.autograd.grad(out, [y, w], g)
    o = r.order.clamp(min=0).long()
    want = torch.where((r.order >= 0)[:, None], g.double()[o // top] * w.detach().double().flatten()[o][:, None], 0.0)
    near(dy, want, (HALF[x.dtype] + 2.0 ** -24) * want.abs() + 1e-7 * (kind == "f16"), "gradient of rows")
    terms = by_token(y.detach(), r.place) * g.double()[:, None]
    near(dw, terms.sum(2), (columns + 1) * 2.0 ** -24 * terms.abs().sum(2), "gradient of weights")
    assert torch.equal(torch.autograd.grad(ops.experts_combine(y, r, w.detach()), y, g)[0], dy)          # one of the two alone
    assert torch.equal(torch.autograd.grad(ops.experts_combine(y.detach(), r, w), w, g)[0], dw)
    plain = ops.experts_combine(y.detach(), r)
    parts = by_token(y.detach(), r.place)
    near(plain, parts.sum(1), (top + 1) * 2.0 ** -24 * parts.abs().sum(1) + HALF[x.dtype] * parts.sum(1).abs(), "combined without weights")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_and_gradients_of_any_strides(kind):
    _, r = routing_of(50, 3, 5)
    for columns in (64, 66, 71):
        x = randn(50, columns + 9, seed=1, kind=kind)[:, 3:3 + columns]
        for v in (x, x.t().contiguous().t(), x[:1].expand(50, columns)):
            leaf = v.detach().requires_grad_()
            xs = ops.experts_gather(leaf, r)
            assert torch.equal(xs.detach(), ops.experts_gather(v.contiguous(), r))
            wide = randn(150, columns + 5, seed=2, kind=kind)
            for g in (wide[:, 5:], wide[:1, 5:].expand(150, columns), wide[:, 5:].t().contiguous().t()):
                assert torch.equal(torch.autograd.grad(xs, leaf, g, retain_graph=True)[0], torch.autograd.grad(xs, leaf, g.contiguous(), retain_graph=True)[0])
            y, w = randn(150, columns + 4, seed=3, kind=kind)[:, 1:1 + columns].requires_grad_(), randn(3, 50, seed=4).t().requires_grad_()
            out = ops.experts_combine(y, r, w)
            want = ops.experts_combine(y.detach().contiguous(), r, w.detach().contiguous())
            assert torch.equal(out.detach(), want)
            g = v[:50]
            for a, b in zip(torch.autograd.grad(out, [y, w], g, retain_graph=True), torch.autograd.grad(out, [y, w], g.contiguous())):
                assert torch.equal(a, b)
    for dtype in (torch.float64, torch.int16, torch.uint8, torch.bool):          # rows of any type are moved
        v = torch.randint(0, 2, (50, 7), device="cuda", generator=gen(1)).to(dtype)
        assert torch.equal(ops.experts_gather(v, r), torch.where((r.order >= 0)[:, None], v[r.order.clamp(min=0).long() // 3], torch.zeros((), device="cuda", dtype=dtype)))


def test_gradients_against_differences():
    ids, r = routing_of(6, 2, 4)
    x, w = randn(6, 5, seed=1).requires_grad_(), randn(6, 2, seed=2).requires_grad_()
    m = randn(12, 5, seed=3)

    def f(x, w):
        return (ops.experts_combine(ops.experts_gather(x, r) * m, r, w) ** 2).sum()
    gx, gw = torch.autograd.grad(f(x, w), [x, w])
    live = torch.where(r.place >= 0, 1.0, 0.0).double()
    mm = by_token(m, r.place)

    def exact(x, w):          # the same in 64 bits, for the differences
        return (((x[:, None] * mm) * (w * live)[..., None]).sum(1) ** 2).sum()
    xd, wd, h = x.detach().double(), w.detach().double(), 1e-6
    for t, g in ((0, gx), (1, gw)):
        for i in range(g.numel()):
            step = torch.zeros(g.numel(), dtype=torch.float64, device="cuda")
            step[i] = h
            step = step.view(g.shape)
            d = (exact(xd + step, wd) - exact(xd - step, wd)) / (2 * h) if t == 0 else (exact(xd, wd + step) - exact(xd, wd - step)) / (2 * h)
            scale = g.abs().max().item()
            assert abs(g.flatten()[i].item() - d.item()) <= 1e-5 * scale + 1e-6          # 32-bit sums of a few terms; differences' own error h^2


# ---------------- together ----------------
def layer(x, ids, weights, w1, w2, experts):
    """A feed-forward of experts as a user writes it: squared relu between two products."""
    r = ops.experts_sort(ids, experts)
    h = ops.experts_product(ops.experts_gather(ops.mx4_quantize(x), r), w1, r.offsets, torch.float32)
    y = ops.experts_product(torch.relu(h) ** 2, w2, r.offsets, torch.float32)
    return ops.experts_combine(y, r, weights)


@pytest.mark.parametrize("tokens", [1, 5, 64, 700])
def test_a_layer_of_experts(tokens):
    E, K, F = 16, 256, 384
    x = randn(tokens, K, seed=1)
    ids = torch.rand(tokens, E, device="cuda", generator=gen(2)).topk(2, 1).indices
    weights = torch.softmax(randn(tokens, 2, seed=3), 1)
    w1, w2 = ops.mx4_quantize(randn(E, F, K, seed=4) * K ** -0.5), ops.mx4_quantize(randn(E, K, F, seed=5) * F ** -0.5)
    got = layer(x, ids, weights, w1, w2, E)
    xv, v1, v2 = quantised(x)[1], values(w1), values(w2)
    want, size = torch.zeros_like(xv), torch.zeros_like(xv)
    for t in range(tokens):
        for j in range(2):
            e = ids[t, j].item()
            # the kernels' own state between the products: another fp32 order of the sums may round a number to the neighbouring code, so the second product is checked on what was quantised
            h = ops.experts_product(x[t:t + 1], ops.Mx4(w1.codes[e:e + 1], w1.scales[e:e + 1], K), torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.float32)
            near(h, xv[t:t + 1] @ v1[e].T, K * 2.0 ** -23 * (xv[t:t + 1].abs() @ v1[e].abs().T), "first product")
            hv = quantised(torch.relu(h) ** 2)[1]
            want[t] += weights[t, j].double() * (hv @ v2[e].T)[0]
            size[t] += weights[t, j].double() * (hv.abs() @ v2[e].abs().T)[0]
        if t > 40:
            break
    n = min(tokens, 42)
    # one token alone takes other kernels than many: where the fp32 sums differ in their last bits, a number on a code's border moves by one code, at most a quarter of its group's largest; allowed in few
    tol = (F + 4) * 2.0 ** -23 * size
    off = ((got.double() - want).abs() > tol)[:n]
    assert off.double().mean() < 0.05, "more than numbers on a border"
    assert ((got.double() - want).abs()[:n] <= tol[:n] + 0.05 * size[:n]).all()


def test_captured_and_replayed():
    E, K, F, T = 8, 160, 96, 30
    x, ids, weights = randn(T, K, seed=1), torch.randint(0, E, (T, 2), device="cuda", generator=gen(2)), torch.softmax(randn(T, 2, seed=3), 1)
    w1, w2 = ops.mx4_quantize(randn(E, F, K, seed=4)), ops.mx4_quantize(randn(E, K, F, seed=5))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x, ids, weights, w1, w2, E)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x, ids, weights, w1, w2, E)
        dense = ops.mx4_product(x, ops.Mx4(w1.codes[0], w1.scales[0], K))
    for seed in (7, 8):
        x.copy_(randn(T, K, seed=seed))
        ids.copy_(torch.randint(-1, E, (T, 2), device="cuda", generator=gen(seed)))
        graph.replay()
        assert torch.equal(out, layer(x, ids, weights, w1, w2, E))
        assert torch.equal(dense, ops.mx4_product(x, ops.Mx4(w1.codes[0], w1.scales[0], K)))


def test_two_streams_at_once():
    """Calls that run at the same time do not share a workspace."""
    w = ops.mx4_quantize(randn(2000, 1024, seed=1))
    xs = [randn(n, 1024, seed=n) for n in (1, 40, 300, 700)]
    want = [ops.mx4_product(x, w) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(ops.mx4_product(x, w))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 4])


def test_refusals():
    w, we = random_mx4(40, 64), random_mx4(3, 40, 64)
    x, off = torch.zeros(5, 64, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    _, r = routing_of(5, 2, 4)
    bad = [
        (lambda: ops.mx4_quantize(x.double()), "float32, bfloat16 or float16"), (lambda: ops.mx4_quantize(x.cpu()), "CUDA tensor"), (lambda: ops.mx4_quantize(x[0, 0]), "columns"),
        (lambda: ops.mx4_read(w, torch.float64), "float32, bfloat16 or float16"), (lambda: ops.mx4_read(w._replace(columns=65)), "uint8 codes"), (lambda: ops.mx4_read(w._replace(scales=w.scales[:39])), "uint8 codes"),
        (lambda: ops.mx4_read(w._replace(codes=w.codes.int())), "uint8 codes"), (lambda: ops.mx4_read(w._replace(codes=w.codes.t().contiguous().t())), "neighbours"),
        (lambda: ops.mx4_read(ops.Mx4(torch.zeros(40, 33, dtype=torch.uint8, device="cuda")[:, 1:], w.scales, 64)), "multiples of 16"),
        (lambda: ops.mx4_product(x, we), "outputs, columns"), (lambda: ops.mx4_product(x[:, :63], w), "63 columns"), (lambda: ops.mx4_product(x.double(), w), "an Mx4"),
        (lambda: ops.mx4_product(x, w, torch.int32), "results are"), (lambda: ops.mx4_product(x.cpu(), w), "CUDA tensor"),
        (lambda: ops.mx4_product(x, w._replace(codes=torch.zeros(40, 40, dtype=torch.uint8, device="cuda")[:, 8:])), "multiples of 16"),
        (lambda: ops.experts_product(x, w, off), "experts, outputs"), (lambda: ops.experts_product(x, we, off[:3]), "offsets"), (lambda: ops.experts_product(x, we, off.long()), "offsets"),
        (lambda: ops.experts_product(x, we, None), "offsets"), (lambda: ops.experts_product(x[None], we, off), "rows, columns"),
        (lambda: ops.experts_sort(x, 4), "int32 or int64"), (lambda: ops.experts_sort(off, 0), "1 to 1024"), (lambda: ops.experts_sort(off, 1025), "1 to 1024"), (lambda: ops.experts_sort(off.view(1, 2, 2), 4), "tokens, top"),
        (lambda: ops.experts_gather(x[:4], r), "4 rows for 5 tokens"), (lambda: ops.experts_gather(x[0], r), "tokens, columns"), (lambda: ops.experts_gather(x, r._replace(order=r.order.long())), "routing"),
        (lambda: ops.experts_gather(x, r._replace(place=r.place[:4])), "routing"), (lambda: ops.experts_gather(x.double().requires_grad_(), r), "gradients"), (lambda: ops.experts_gather(we, r), "Mx4 of"),
        (lambda: ops.experts_combine(x, r), "y is"), (lambda: ops.experts_combine(torch.zeros(10, 4, device="cuda").double(), r), "y is"),
        (lambda: ops.experts_combine(torch.zeros(10, 4, device="cuda"), r, torch.zeros(2, 5, device="cuda")), "weights"), (lambda: ops.experts_combine(torch.zeros(10, 4, device="cuda"), r, off), "weights"),
    ]
    for f, text in bad:
        with pytest.raises(NB200Error, match=text):
            f()
    with pytest.raises(RuntimeError):          # no gradient of a gradient
        y = x.clone().requires_grad_()
        g, = torch.autograd.grad((ops.experts_gather(y, r) ** 2).sum(), y, create_graph=True)
        torch.autograd.grad(g.sum(), y)


# ---------------- further sizes, strides and orders of calls ----------------
@pytest.mark.parametrize("rows,outputs,columns", [(3001, 4000, 1000), (1024, 9728, 256), (2048, 5001, 777), (700, 20000, 96), (4096, 2600, 3333)])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_large_products(rows, outputs, columns, kind):
    """Many tiles: shared by two blocks, and by one, with outputs that end inside a tile."""
    x, w = random_mx4(rows, columns, seed=rows), random_mx4(outputs, columns, seed=3)
    x.scales.clamp_(max=129)          # (sums within fp16)
    w.scales.sub_(5)
    check_product(x, w, DT[kind])


@pytest.mark.parametrize("counts", [[700, 0, 255, 1, 256, 257] * 3, [5000, 1, 0, 3], [300] * 40])
def test_large_products_of_experts(counts):
    x, w = random_mx4(sum(counts) + 7, 512, seed=1), random_mx4(len(counts), 1000, 512, seed=2)
    check_product(x, w, torch.bfloat16, offsets_of(counts))
    got = check_product(x, w, torch.float32, offsets_of(counts, first=7))
    assert (got[:7] == 0).all()


@pytest.mark.parametrize("rows", [1, 3, 6, 18, 200])
@pytest.mark.parametrize("columns", [189, 191, 61, 1])
def test_what_fills_up_a_group_does_not_count(rows, columns):
    """Rows of an odd number of columns out of longer ones: the rest of the last group, and of its last byte, holds other numbers."""
    G = -(-columns // 32)
    x, w = random_mx4(rows, 512, seed=5), random_mx4(130, 512, seed=6)
    a, b = ops.Mx4(x.codes[:, :16 * G], x.scales[:, :G], columns), ops.Mx4(w.codes[:, :16 * G], w.scales[:, :G], columns)
    check_product(a, b, torch.float32)
    we = ops.Mx4(b.codes.expand(2, 130, 16 * G), b.scales.expand(2, 130, G), columns)          # one matrix for all experts
    check_product(a, we, torch.float32, offsets_of([rows // 2, rows - rows // 2]))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 2, 4, 6, 16, 17, 40])
@pytest.mark.parametrize("offset,columns", [(0, 640), (1, 640), (3, 517), (8, 96), (2, 2500)])
def test_products_of_rows_of_numbers_anywhere(kind, rows, offset, columns):
    big = randn(rows, columns + offset + 5, seed=rows, kind=kind)
    big[:, :offset] = math.nan
    big[:, offset + columns:] = math.nan
    w = ops.mx4_quantize(randn(300, columns, seed=2))
    x = big[:, offset:offset + columns]
    got = check_product(x, w, torch.float32)
    assert torch.equal(got, ops.mx4_product(ops.mx4_quantize(x), w, torch.float32)) or columns == 2500          # (a depth may be split otherwise)
    check_product(x.t().contiguous().t(), w, torch.float32)
    check_product(x[:1].expand(rows, columns), w, torch.float32)


def test_one_row_of_a_tensor_of_any_stride():
    """The stride of a single row is of no account."""
    K = 300
    x, w = random_mx4(1, K, seed=1), random_mx4(1, K, seed=2)

    def odd(m):
        codes, scales = (torch.empty(1000, dtype=torch.uint8, device="cuda").as_strided(t.shape, (7, 1)) for t in (m.codes, m.scales))
        codes.copy_(m.codes), scales.copy_(m.scales)
        return ops.Mx4(codes, scales, K)
    near(ops.mx4_read(odd(x)), values(x).float(), 0.0, "read")
    check_product(odd(x), odd(w), torch.float32)
    check_product(odd(x), random_mx4(50, K, seed=3), torch.float32)
    one = ops.Mx4(odd(w).codes[None], odd(w).scales[None], K)
    check_product(odd(x), one, torch.float32, offsets_of([1]))


@pytest.mark.parametrize("rows", [1, 20, 300])
def test_products_of_small_and_large_scales(rows):
    """Numbers from 2^-100 to 2^100 in one product, each output of one size."""
    x, w = random_mx4(rows, 96, seed=1), random_mx4(201, 96, seed=2)
    w.scales[:] = torch.arange(27, 228, device="cuda").to(torch.uint8)[:, None]
    check_product(x, w, torch.float32)


def test_sort_of_many_places_and_experts():
    ids = torch.randint(0, 1100, (20000, 5), device="cuda", generator=gen(1))
    for a, b in zip(ops.experts_sort(ids, 1024), sorted_reference(ids, 1024)):
        assert torch.equal(a.cpu(), b)


def state_of_all(seed):
    s = dict(x=randn(40, 200, seed=seed), big=randn(600, 512, seed=seed, kind="bf16"), ids=torch.randint(-1, 6, (40, 3), device="cuda", generator=gen(seed)), weights=torch.softmax(randn(40, 3, seed=seed), 1))
    s["w"], s["wide"], s["we"] = ops.mx4_quantize(randn(300, 200, seed=seed)), ops.mx4_quantize(randn(20000, 512, seed=seed)), ops.mx4_quantize(randn(6, 200, 200, seed=seed))
    return s


def run_of_all(s):
    r = ops.experts_sort(s["ids"], 6)
    y = ops.experts_product(ops.experts_gather(s["x"], r), s["we"], r.offsets)
    return [*r, y, ops.experts_combine(y, r, s["weights"]), ops.mx4_product(s["x"][:2], s["w"]), ops.mx4_product(s["x"], s["w"]), ops.mx4_product(ops.mx4_quantize(s["x"]), s["w"]),
            ops.mx4_product(s["big"], s["wide"]), ops.mx4_read(ops.mx4_quantize(s["x"][:, 1:]))]


def test_two_graphs_that_share_memory():
    a, b = state_of_all(21), state_of_all(22)
    want = [[t.clone() for t in run_of_all(s)] for s in (a, b)]
    torch.cuda.synchronize()
    graphs, outs, pool = [], [], torch.cuda.graph_pool_handle()
    for s in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(run_of_all(s))
        graphs.append(graph)
    for i in (0, 1, 1, 0, 1):
        graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(outs[i], want[i]))
        assert torch.equal(run_of_all(a)[4], want[0][4])


def test_all_on_four_streams_at_once():
    states = [state_of_all(30 + i) for i in range(4)]
    want = [[t.clone() for t in run_of_all(s)] for s in states]
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for s, stream in zip(states, streams):
            with torch.cuda.stream(stream):
                got.append(run_of_all(s))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(g, w))


def test_a_captured_step_that_learns():
    """Forward and backward in one graph, as a training loop captures them."""
    x, w = randn(64, 96, seed=1).requires_grad_(), randn(64, 2, seed=2).requires_grad_()
    ids = torch.randint(0, 5, (64, 2), device="cuda", generator=gen(3))

    def step():
        r = ops.experts_sort(ids, 5)
        out = ops.experts_combine(torch.tanh(ops.experts_gather(x, r)), r, w)
        return torch.autograd.grad(out.square().sum(), [x, w])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (5, 6):
        with torch.no_grad():
            x.copy_(randn(64, 96, seed=seed))
        ids.copy_(torch.randint(-1, 5, (64, 2), device="cuda", generator=gen(seed)))
        graph.replay()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_a_routing_changed_in_between_is_noticed():
    _, r = routing_of(8, 2, 4)
    x = randn(8, 16).requires_grad_()
    xs = ops.experts_gather(x, r)
    r.place.fill_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(xs, x, torch.ones_like(xs))


FIRST_CALLS = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import torch
import test_gpu_mx4_experts as t
s = t.state_of_all(1)
ids = torch.randint(0, 1000, (20000, 4), device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = t.run_of_all(s) + list(t.ops.experts_sort(ids, 1000))
graph.replay()
torch.cuda.synchronize()
want = t.run_of_all(s) + list(t.ops.experts_sort(ids, 1000))
assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(out, want))
print("the same")
"""


def test_the_first_calls_of_a_process_may_be_captured():
    here = os.path.dirname(os.path.abspath(__file__))
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(root=os.path.dirname(here), tests=here)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "the same" in done.stdout, done.stderr[-2000:]


# ---------------- what a backward pass keeps, and what it cannot give ----------------
def test_combine_keeps_what_its_gradients_need():
    """Rows that nothing is multiplied with may change before the backward pass, weights too where only theirs is wanted; what a wanted gradient reads may not."""
    ids = torch.tensor([[0, 3], [1, -1], [2, 0]], device="cuda")
    r = ops.experts_sort(ids, 4)
    y0, w0, g = torch.randn(6, 24, device="cuda"), torch.rand(3, 2, device="cuda"), torch.randn(3, 24, device="cuda")

    def run(y_grad, w_grad, change):
        leaf, weights = y0.clone().requires_grad_(y_grad), w0.clone().requires_grad_(w_grad)
        y, w = leaf * 1, weights * 1
        out = ops.experts_combine(y, r, w)
        with torch.no_grad():
            for name in change:
                {"y": y, "w": w}[name].zero_()
        out.backward(g)
        return leaf.grad, weights.grad

    dy, dw = run(True, True, "")
    known = (r.order >= 0)[:, None]
    assert torch.equal(dy, torch.where(known, g[r.order.long().clamp(min=0) // 2] * w0.flatten()[r.order.long().clamp(min=0)][:, None], 0))
    only_y, none = run(True, False, "y")
    assert torch.equal(only_y, dy) and none is None
    none, only_w = run(False, True, "w")
    assert torch.equal(only_w, dw) and none is None
    for kinds, change in (((True, True), "y"), ((True, True), "w"), ((True, False), "w"), ((False, True), "y")):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            run(*kinds, change)


def test_no_gradients_of_gradients():
    """A graph of the gradient is refused where the gradient depends on something that has one: it would be lost."""
    ids = torch.tensor([[0, 3], [1, -1], [2, 0]], device="cuda")
    r = ops.experts_sort(ids, 4)
    y, w = torch.randn(6, 24, device="cuda", requires_grad=True), torch.rand(3, 2, device="cuda", requires_grad=True)
    for leaf in (y, w):
        with pytest.raises(NB200Error, match="gradients of gradients"):
            torch.autograd.grad(ops.experts_combine(y, r, w).sum(), leaf, create_graph=True)
    g, = torch.autograd.grad(ops.experts_combine(y, r, w.detach()).sum(), y, create_graph=True)          # of y's nothing depends on y
    want, = torch.autograd.grad(ops.experts_combine(y, r, w.detach()).sum(), y)
    assert torch.equal(g, want) and not g.requires_grad
    x = torch.randn(3, 24, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(ops.experts_gather(x, r).sum(), x, create_graph=True)
    assert torch.equal(g, torch.tensor([2.0, 1.0, 2.0], device="cuda")[:, None].expand(3, 24))


def test_arguments_of_other_kinds_are_refused():
    x = torch.zeros(3, 64, device="cuda")
    w, ids = ops.mx4_quantize(x), torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    for f in (lambda: ops.mx4_read(x), lambda: ops.mx4_product(x, x), lambda: ops.mx4_product(w, tuple(w)), lambda: ops.experts_product(x, x[None], torch.tensor([0, 3], dtype=torch.int32, device="cuda"))):
        with pytest.raises(NB200Error, match="is an Mx4"):
            f()
    for f in (lambda: ops.experts_gather(x, ids), lambda: ops.experts_gather(w, ids), lambda: ops.experts_combine(torch.zeros(6, 4, device="cuda"), tuple(ops.experts_sort(ids, 2)))):
        with pytest.raises(NB200Error, match="what experts_sort gives"):
            f()


@pytest.mark.parametrize("blocks", [1, 2, 4, 8, 16])
def test_sort_at_the_borders_of_blocks(blocks):
    """Lists of just as many places as so many blocks take, and one more or less; of one expert, and of many."""
    for n in (1024 * blocks - 1, 1024 * blocks, 1024 * blocks + 1):
        for experts in (1, 33, 1024):
            ids = torch.randint(-1, experts + 1, (n,), device="cuda", generator=torch.Generator("cuda").manual_seed(n))
            for a, b in zip(ops.experts_sort(ids, experts), sorted_reference(ids, experts)):
                assert torch.equal(a.cpu(), b.reshape(a.shape)), (n, experts)


def test_no_derivatives_in_forward_mode():
    """A tangent that comes in, with an input or with a gradient on its way back, is refused: it would be lost.  Inputs without one go on inside a level too."""
    forward = torch.autograd.forward_ad
    ids = torch.tensor([[0, 3], [1, -1], [2, 0]], device="cuda")
    r = ops.experts_sort(ids, 4)
    x, y, w = randn(3, 24, seed=1), randn(6, 24, seed=2), randn(3, 2, seed=3)
    leaf = x.clone().requires_grad_()
    rows, weights = y.clone().requires_grad_(), w.clone().requires_grad_()
    with forward.dual_level():
        def dual(t):
            return forward.make_dual(t, torch.ones_like(t))
        refused = [lambda: ops.experts_gather(dual(x), r), lambda: ops.experts_gather(dual(x.double()), r), lambda: ops.experts_gather(dual(leaf), r), lambda: ops.experts_combine(dual(y), r), lambda: ops.experts_combine(dual(y), r, w),
                   lambda: ops.experts_combine(y, r, dual(w)), lambda: ops.experts_combine(rows, r, dual(w)), lambda: ops.experts_combine(y, r, dual(w.double())), lambda: torch.autograd.grad(ops.experts_gather(leaf, r), leaf, dual(y)),
                   lambda: torch.autograd.grad(ops.experts_combine(rows, r, weights), rows, dual(x)), lambda: torch.autograd.grad(ops.experts_combine(rows, r, weights), weights, dual(x))]
        for f in refused:
            with pytest.raises(NB200Error, match="forward mode"):
                f()
            with torch.no_grad(), pytest.raises(NB200Error, match="forward mode"):          # (which is not what forward mode goes by)
                refused[0]()
        inside = ops.experts_gather(x, r), ops.experts_combine(y, r, w), torch.autograd.grad(ops.experts_combine(rows, r, weights).sum(), [rows, weights])
    assert torch.equal(inside[0], ops.experts_gather(x, r)) and torch.equal(inside[1], ops.experts_combine(y, r, w))
    for a, b in zip(inside[2], torch.autograd.grad(ops.experts_combine(rows, r, weights).sum(), [rows, weights])):
        assert torch.equal(a, b)
    with pytest.raises(NB200Error, match="forward mode"):
        torch.func.jvp(lambda v: ops.experts_gather(v, r), (x,), (torch.ones_like(x),))


def test_conjugated_and_negated_views():
    """Views whose numbers are not yet what they stand for in memory."""
    ids = torch.tensor([[0, 3], [1, -1], [2, 0]], device="cuda")
    r = ops.experts_sort(ids, 4)
    x, y, w, g = randn(3, 96, seed=1), randn(6, 96, seed=2), randn(3, 2, seed=3), randn(3, 96, seed=4)
    m, me = ops.mx4_quantize(randn(40, 96, seed=5)), ops.mx4_quantize(randn(4, 40, 96, seed=6))
    neg = torch._neg_view
    assert neg(x).is_neg() and neg(x).is_contiguous()
    z = torch.complex(x, x.flip(0))
    for v in (z.conj(), z.conj()[:, 3:90], neg(z.conj())):
        assert torch.equal(ops.experts_gather(v, r), ops.experts_gather(v.clone().resolve_conj().resolve_neg(), r))
    assert torch.equal(ops.experts_gather(z.conj(), r)[0], z[0].conj().resolve_conj())
    for a, b in ((neg(x), -x), (neg(x)[:, 3:77], -x[:, 3:77]), (neg(x[0]), -x[0]), (neg(x).view(3, 2, 48), -x.view(3, 2, 48))):
        assert all(torch.equal(s, t) for s, t in zip(ops.mx4_quantize(a)[:2], ops.mx4_quantize(b)[:2]))
    for f in (lambda v: ops.mx4_product(v, m), lambda v: ops.experts_gather(v, r)):
        assert torch.equal(f(neg(x)), f(-x))
    assert torch.equal(ops.experts_product(neg(y), me, r.offsets), ops.experts_product(-y, me, r.offsets))
    want = ops.experts_combine(-y, r, -w)
    assert torch.equal(ops.experts_combine(neg(y), r, neg(w)), want) and torch.equal(ops.experts_combine(neg(y), r, neg(w.double())), ops.experts_combine(-y, r, -w.double()))
    leaf, weights = y.clone().requires_grad_(), w.clone().requires_grad_()
    for a, b in zip(torch.autograd.grad(ops.experts_combine(neg(leaf), r, neg(weights)), [leaf, weights], neg(g)), torch.autograd.grad(ops.experts_combine(-leaf, r, -weights), [leaf, weights], -g)):
        assert torch.equal(a, b)
    leaf = x.clone().requires_grad_()
    for a, b in zip(torch.autograd.grad(ops.experts_gather(neg(leaf), r), leaf, neg(y)), torch.autograd.grad(ops.experts_gather(-leaf, r), leaf, -y)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("columns", [1, 7, 36, 267, 1001])
def test_gradient_of_rows_alone_at_odd_widths(kind, columns):
    """Rows that start anywhere, their gradient among NaN: without the weights' gradient y is not there to be read."""
    _, r = routing_of(90, 3, 5, seed=columns)
    wide = torch.full((90, columns + 9), math.nan, device="cuda", dtype=DT[kind])
    g, w = wide[:, 5:5 + columns], randn(90, 2 + 1, seed=2)
    g.copy_(randn(90, columns, seed=1, kind=kind))
    y = randn(270, columns, seed=3, kind=kind).requires_grad_()
    o = r.order.clamp(min=0).long()
    for weights in (w, None):
        dy, = torch.autograd.grad(ops.experts_combine(y, r, weights), y, g)
        factor = torch.ones(270, device="cuda") if weights is None else w.flatten()[o]
        want = torch.where((r.order >= 0)[:, None], (g.float()[o // 3] * factor[:, None]).to(y.dtype), torch.zeros((), device="cuda", dtype=y.dtype))
        assert torch.equal(dy, want)          # (one product in 32 bits, rounded once)


@pytest.mark.parametrize("columns", [1, 33, 70, 160, 1000])
@pytest.mark.parametrize("dropped", [0.0, 0.3, 1.0])
def test_gather_of_rows_in_4_bits(columns, dropped):
    """Codes and scales of odd numbers of groups, out of wider rows too, and places without an expert: those stand for zeros."""
    G = -(-columns // 32)
    for tokens, top in ((1, 1), (37, 3), (500, 2)):
        _, r = routing_of(tokens, top, 9, seed=tokens, dropped=dropped)
        wide = random_mx4(tokens, 32 * (G + 3), seed=columns)
        live, o = (r.order >= 0)[:, None], r.order.clamp(min=0).long() // top
        for x in (random_mx4(tokens, columns, seed=columns), ops.Mx4(wide.codes[:, 16:16 + 16 * G], wide.scales[:, 1:1 + G], columns)):
            got = ops.experts_gather(x, r)
            assert got.columns == columns and torch.equal(got.codes, torch.where(live, x.codes[o], 0)) and torch.equal(got.scales, torch.where(live, x.scales[o], 0))
            near(ops.mx4_read(got), torch.where(live, values(x)[o], 0.0).float(), 0.0, "gathered")


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 2, 4, 6, 16, 17, 40])
def test_deep_rows_quantised_on_the_way_and_before(rows, kind):
    """The two may share the depth out otherwise.  An instruction adds two groups' sums to what is there, three roundings of at most 2^-23 of the magnitudes' sum S; a depth of 2500 is 40 instructions and at
    most 8 parts: either side is off by (3 x 40 + 8) 2^-23 S."""
    K = 2500
    x, w = randn(rows, K, seed=rows, kind=kind), ops.mx4_quantize(randn(300, K, seed=2))
    size = quantised(x)[1].abs() @ values(w).abs().T
    near(ops.mx4_product(x, w, torch.float32), ops.mx4_product(ops.mx4_quantize(x), w, torch.float32), 2 * (3 * 40 + 8) * 2.0 ** -23 * size, "quantised on the way")


def test_which_calls_carry_gradients():
    """Rows in 4 bits and their products carry none; a gradient that is to pass them is the caller's to give."""
    x, w = randn(5, 64, seed=1).requires_grad_(), randn(2, 40, 64, seed=2).requires_grad_()
    m = ops.mx4_quantize(w)
    r = ops.experts_sort(torch.tensor([0, 1, 1, -1, 0], device="cuda"), 2)
    rows = ops.experts_gather(x, r)
    assert rows.requires_grad and ops.experts_combine(rows, r).requires_grad
    y = ops.experts_product(rows, m, r.offsets)
    assert not any(t.requires_grad for t in (m.codes, m.scales, ops.mx4_read(m), ops.mx4_product(x, ops.Mx4(m.codes[0], m.scales[0], 64)), y))
    weights = torch.rand(5, device="cuda").requires_grad_()
    g, = torch.autograd.grad(ops.experts_combine(y, r, weights).sum(), weights)          # those of the weights go by the rows as they are
    near(g, by_token(y, r.place).sum(-1), (40 + 1) * 2.0 ** -24 * by_token(y, r.place).abs().sum(-1), "gradient of weights")


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,outputs,columns", [(1, 9728, 2561), (1, 9728, 2816), (2, 5000, 2999), (4, 9728, 3328), (5, 300, 3327), (1, 9728, 3329), (5, 2000, 3329), (1, 19500, 3328), (3, 9728, 6656), (1, 9728, 6657), (1, 9728, 7000)])
def test_few_rows_as_deep_as_a_block_has_room_for(kind, rows, outputs, columns):
    x = randn(rows, columns + 3, seed=rows, kind=kind)[:, 3:]
    check_product(x, ops.mx4_quantize(randn(outputs, columns, seed=2)), torch.float32)
    if rows > 1:
        w = ops.mx4_quantize(randn(3, 500, columns, seed=3))
        check_product(x, w, torch.float32, offsets_of([1, 0, rows - 1]))
