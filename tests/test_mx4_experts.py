"""CPU tests of products in microscaled 4-bit floating point and of routed experts: what their C entry points refuse before any device is looked for, and that there is no CPU fallback."""
import ctypes as C

import pytest

from nano_b200 import engine as E

EINVAL, ENODEV = -1, -3
P = 4096          # an address that is never followed: every call here is refused first


def refused(rc, text):
    assert rc == EINVAL, (rc, E.lib().nb200_last_error())
    assert text in E.lib().nb200_last_error().decode(), E.lib().nb200_last_error()


def rows(**kw):
    base = dict(codes=P, scales=P, code_stride=64, scale_stride=4, x=P, x_stride=128, type=1, rows=3, columns=128)
    base.update(kw)
    return C.byref(E.Mx4Rows(**base))


@pytest.mark.parametrize("call", ["nb200_dev_mx4_quantize", "nb200_dev_mx4_read"])
def test_rows_refusals(call):
    f = getattr(E.lib(), call)
    refused(f(None, None), "null")
    refused(f(rows(type=3), None), "fp32, bf16 or fp16")
    refused(f(rows(columns=0), None), "no numbers")
    refused(f(rows(columns=1 << 31), None), "too long")
    for name in ("codes", "scales", "x"):
        refused(f(rows(**{name: None}), None), "null")
    refused(f(rows(codes=P + 8), None), "multiples of 16")
    refused(f(rows(code_stride=72), None), "multiples of 16")
    refused(f(rows(code_stride=48), None), "overlap")
    refused(f(rows(scale_stride=3), None), "overlap")
    refused(f(rows(columns=129), None), "overlap")
    refused(f(rows(x=P + 1), None), "aligned")
    assert f(rows(rows=0), None) == 0
    if call == "nb200_dev_mx4_read":
        refused(f(rows(x_stride=127), None), "overlap")


def product(**kw):
    base = dict(x=P, x_scales=P, x_stride=64, xs_stride=4, w=P, w_scales=P, w_stride=64, ws_stride=4, w_expert=0, ws_expert=0, out=P, out_stride=100, offsets=None,
                x_type=3, out_type=1, rows=5, outputs=100, columns=128, experts=0)
    base.update(kw)
    return C.byref(E.Mx4Product(**base))


def test_product_refusals():
    L, need = E.lib(), C.c_uint64(7)
    for f in (lambda p: L.nb200_dev_mx4_product(p, P, 1 << 40, None), lambda p: L.nb200_dev_mx4_product_workspace(p, C.byref(need))):
        refused(f(None), "null")
        refused(f(product(x_type=4)), "rows are fp32, bf16, fp16")
        refused(f(product(out_type=3)), "results are fp32")
        for name in ("rows", "outputs", "columns"):
            refused(f(product(**{name: (1 << 30) + 1})), "too large")
        refused(f(product(experts=1025)), "at most 1024")
        refused(f(product(columns=0)), "no numbers")
        for name in ("x", "x_scales", "w", "w_scales", "out"):
            refused(f(product(**{name: None})), "null")
        refused(f(product(experts=2)), "null")
        refused(f(product(w=P + 8)), "multiples of 16")
        refused(f(product(w_stride=72)), "multiples of 16")
        refused(f(product(w_expert=8, experts=2, offsets=P)), "multiples of 16")
        refused(f(product(x=P + 4)), "multiples of 16")
        refused(f(product(x_stride=68)), "multiples of 16")
        refused(f(product(w_stride=1 << 38)), "2^38")
        refused(f(product(w_stride=48)), "overlap")
        refused(f(product(x_stride=48)), "overlap")
        refused(f(product(x_type=0, x=P + 2)), "aligned")
        refused(f(product(out=P + 1)), "aligned")
        refused(f(product(out_stride=99)), "overlap")
        refused(f(product(experts=2, offsets=P + 2)), "aligned")
        assert f(product(rows=0)) == 0 and f(product(outputs=0)) == 0
    refused(L.nb200_dev_mx4_product_workspace(product(), None), "null")
    assert L.nb200_dev_mx4_product_workspace(product(), C.byref(need)) == 0 and need.value == 0
    assert L.nb200_dev_mx4_product_workspace(product(x_type=1), C.byref(need)) == 0 and need.value == 0          # few rows are quantised on the way
    assert L.nb200_dev_mx4_product_workspace(product(x_type=1, columns=100, rows=5000), C.byref(need)) == 0 and need.value >= 5000 * 4 * 17
    n, text = need.value, "%d are needed" % need.value
    refused(L.nb200_dev_mx4_product(product(x_type=1, columns=100, rows=5000), P, n - 1, None), text)
    refused(L.nb200_dev_mx4_product(product(x_type=1, columns=100, rows=5000), None, n, None), text)
    refused(L.nb200_dev_mx4_product(product(x_type=1, columns=100, rows=5000), P + 8, n, None), text)


def sort(order=P, offsets=P, place=P, ids=P, id_bytes=8, n=10, experts=4):
    return E.lib().nb200_dev_experts_sort(order, offsets, place, ids, id_bytes, n, experts, None)


def gather(out=P, out_stride=64, x=P, x_stride=64, row_bytes=64, order=P, n=10, top=2, tokens=5):
    return E.lib().nb200_dev_experts_gather(out, out_stride, x, x_stride, row_bytes, order, n, top, tokens, None)


def test_sort_and_gather_refusals():
    refused(sort(experts=0), "1 to 1024")
    refused(sort(experts=1025), "1 to 1024")
    refused(sort(n=(1 << 30) + 1), "too many")
    refused(sort(id_bytes=2), "32-bit or 64-bit")
    for name in ("order", "offsets", "place", "ids"):
        refused(sort(**{name: None}), "null")
    refused(sort(ids=P + 4), "aligned")
    refused(sort(order=P + 2), "aligned")
    refused(gather(n=(1 << 30) + 1), "too many")
    refused(gather(row_bytes=(1 << 30) + 1), "too many")
    for name in ("out", "x", "order"):
        refused(gather(**{name: None}), "null")
    refused(gather(top=0), "null")
    refused(gather(order=P + 1), "aligned")
    refused(gather(out_stride=63), "overlap")
    assert gather(n=0) == 0 and gather(row_bytes=0) == 0


def combined(**kw):
    base = dict(out=P, out_stride=64, y=P, y_stride=64, weights=P, place=P, order=P, type=1, tokens=5, top=2, rows=10, columns=64, grad=P, grad_stride=64, dy=P, dy_stride=64, dweights=P)
    base.update(kw)
    return C.byref(E.ExpertsRows(**base))


def test_combine_refusals():
    L = E.lib()
    for f in (lambda p: L.nb200_dev_experts_combine(p, None), lambda p: L.nb200_dev_experts_combine_grad(p, None)):
        refused(f(None), "null")
        refused(f(combined(type=3)), "fp32, bf16 or fp16")
        refused(f(combined(tokens=1 << 30)), "too many")
        refused(f(combined(rows=(1 << 30) + 1)), "too many")
        refused(f(combined(columns=(1 << 30) + 1)), "too many")
        refused(f(combined(y=P + 1)), "aligned")
        refused(f(combined(weights=P + 2)), "aligned")
        refused(f(combined(place=None)), "null")
        refused(f(combined(y=None)), "null")
        assert f(combined(tokens=0, rows=0)) == 0
    refused(L.nb200_dev_experts_combine(combined(out=None), None), "null")
    refused(L.nb200_dev_experts_combine(combined(out_stride=63), None), "overlap")
    refused(L.nb200_dev_experts_combine_grad(combined(order=None), None), "null")
    refused(L.nb200_dev_experts_combine_grad(combined(grad=None), None), "null")
    refused(L.nb200_dev_experts_combine_grad(combined(rows=11), None), "11 rows of 10 places")
    refused(L.nb200_dev_experts_combine_grad(combined(dy_stride=63), None), "overlap")
    assert L.nb200_dev_experts_combine_grad(combined(dy=None, dweights=None), None) == 0


@pytest.mark.skipif(E.device_count() > 0, reason="box has a GPU")
def test_no_cpu_fallback():
    L = E.lib()
    assert L.nb200_dev_mx4_quantize(rows(), None) == ENODEV and L.nb200_dev_mx4_read(rows(), None) == ENODEV
    assert L.nb200_dev_mx4_product(product(), None, 0, None) == ENODEV
    assert sort() == ENODEV and gather() == ENODEV
    assert L.nb200_dev_experts_combine(combined(), None) == ENODEV and L.nb200_dev_experts_combine_grad(combined(), None) == ENODEV
    from nano_b200 import ops
    import torch
    for f in (lambda: ops.mx4_quantize(torch.zeros(2, 32)), lambda: ops.mx4_read(ops.Mx4(torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(2, 1, dtype=torch.uint8), 32)),
              lambda: ops.experts_sort(torch.zeros(2, 2, dtype=torch.int64), 4), lambda: ops.experts_gather(torch.zeros(2, 4), ops.Routing(*[torch.zeros(4, dtype=torch.int32)] * 3)),
              lambda: ops.experts_combine(torch.zeros(2, 4), ops.Routing(*[torch.zeros(4, dtype=torch.int32)] * 3))):
        with pytest.raises(E.NB200Error, match="CUDA tensor"):
            f()


def test_gradient_of_weights_wants_order_whatever_the_columns():
    """The kernel reads order for every row, of rows without columns too; without rows it reads none."""
    call = E.lib().nb200_dev_experts_combine_grad
    none = dict(columns=0, dy=None, dy_stride=0, grad=None, y=None)
    refused(call(combined(order=None, **none), None), "null")
    refused(call(combined(place=None, **none), None), "null")
    refused(call(combined(order=None, dy=None), None), "null")
    if E.device_count() <= 0:          # (these would be launched)
        assert call(combined(**none), None) == ENODEV
        assert call(combined(order=None, rows=0, **none), None) == ENODEV


def test_one_row_needs_no_workspace_up_to_the_room_of_a_block():
    """Thirteen steps of 256 columns, twice as many where two blocks share them: at no depth below that is a launch put before the product."""
    need = C.c_uint64(7)
    for kind in (0, 1, 2):
        for outputs in (1, 1000, 9728, 128 * 148):
            for columns in range(32, 6656 + 1, 32):
                groups = columns // 32
                p = product(x_type=kind, x_scales=None, x_stride=columns, columns=columns, rows=1, outputs=outputs, w_stride=16 * groups, ws_stride=groups, out_stride=outputs)
                assert E.lib().nb200_dev_mx4_product_workspace(p, C.byref(need)) == 0 and need.value == 0, (kind, outputs, columns)
