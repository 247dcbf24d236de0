"""CPU tests of the operators on device memory: what their C entry points refuse, before any device is looked for, and that there is no CPU fallback."""
import ctypes as C
import os
import re

import numpy as np
import pytest

from conftest import ROOT
from nano_b200 import engine as E

EINVAL, ENODEV = -1, -3
P = 4096          # an address that is never followed: every call here is refused first


def refused(rc, text):
    assert rc == EINVAL, (rc, E.lib().nb200_last_error())
    assert text in E.lib().nb200_last_error().decode()


def logprobs(logits=P, kind=0, stride=100, rows=2, vocab=100, tokens=P, token_bytes=8, top=0, lp=P, ent=P, top_lp=P, top_id=P):
    return E.lib().nb200_dev_token_logprobs(lp, ent, top_lp, top_id, logits, kind, stride, rows, vocab, tokens, token_bytes, top, None)


def test_logprobs_refusals():
    refused(logprobs(kind=3), "fp32, bf16 or fp16")
    refused(logprobs(logits=None), "bad logits")
    refused(logprobs(vocab=0), "bad logits")
    refused(logprobs(vocab=1 << 31), "bad logits")
    refused(logprobs(logits=P + 2), "aligned")
    refused(logprobs(logits=P + 1, kind=1), "aligned")
    refused(logprobs(tokens=P + 4), "aligned")
    refused(logprobs(token_bytes=2), "32-bit or 64-bit")
    refused(logprobs(top=33), "at most 32")
    refused(logprobs(vocab=4, top=5), "no more than the vocabulary")
    refused(logprobs(tokens=None), "need tokens")


def pages(pools, src, dst, n_pages=10, size=64, stride=64):
    n = len(pools)
    src, dst = np.asarray(src, np.uint32), np.asarray(dst, np.uint32)
    return E.lib().nb200_dev_pages_copy((C.c_void_p * n)(*pools), (C.c_uint64 * n)(*[size] * n), (C.c_uint64 * n)(*[stride] * n), (C.c_uint32 * n)(*[n_pages] * n), n,
                                        E._p(src, E.u32p), E._p(dst, E.u32p), src.size, None)


def test_pages_copy_refusals():
    refused(pages([P], [10], [0]), "the smallest pool has 10")
    refused(pages([P], [0], [10]), "the smallest pool has 10")
    refused(pages([P], [0, 1], [2, 2]), "written twice")
    refused(pages([P], [0, 1], [1, 2]), "written and read")
    refused(pages([P], [3], [3]), "written and read")
    refused(pages([P, 0], [0], [1]), "pool 1 is null")
    refused(pages([P], [0], [1], size=64, stride=32), "pages of 64 bytes every 32")
    assert pages([P], [], []) == 0          # nothing to do
    assert pages([], [], []) == 0


def rows(**kw):
    base = dict(pool=P, page_stride=8 * 40 * 128, n_pages=4, kv_heads=8, head_dim=128, type=1, tokens=3, slots=P, k=P, v=P, k_token=1024, k_head=128, v_token=1024, v_head=128)
    base.update(kw)
    return C.byref(E.Kv4Rows(**base))


@pytest.mark.parametrize("call", ["nb200_dev_kv4_write", "nb200_dev_kv4_read"])
def test_rows_refusals(call):
    f = getattr(E.lib(), call)
    refused(f(None, None), "null")
    refused(f(rows(head_dim=48), None), "multiples of 32")
    refused(f(rows(head_dim=288), None), "multiples of 32")
    refused(f(rows(head_dim=0), None), "multiples of 32")
    refused(f(rows(kv_heads=0), None), "kv_heads")
    refused(f(rows(n_pages=1 << 27), None), "32-bit")
    refused(f(rows(pool=P + 8), None), "multiples of 16")
    refused(f(rows(page_stride=8 * 40 * 128 + 8), None), "multiples of 16")
    refused(f(rows(page_stride=7 * 40 * 128), None), "overlap")
    refused(f(rows(pool=None), None), "null pool")
    refused(f(rows(type=3), None), "fp32, bf16 or fp16")
    refused(f(rows(slots=None), None), "null")
    refused(f(rows(k=None), None), "null")
    refused(f(rows(k=P + 1), None), "aligned")
    refused(f(rows(slots=P + 2), None), "aligned")
    refused(f(rows(tokens=(1 << 32) - 1, kv_heads=65535, page_stride=65535 * 40 * 128), None), "too many")
    assert f(rows(tokens=0), None) == 0


def attention(**kw):
    base = dict(q=P, out=P, q_batch=2048, q_token=2048, q_head=128, o_batch=2048, o_token=2048, o_head=128, pool=P, page_stride=8 * 40 * 128, n_pages=4, kv_heads=8, head_dim=128, type=1,
                batch=2, tokens=1, heads=16, width=2, table_stride=2, table=P, lens=P, sinks=None, scale=0.1, softcap=0.0, window=0, block=0)
    base.update(kw)
    return C.byref(E.Kv4Attention(**base))


def test_attention_refusals():
    L, need = E.lib(), C.c_uint64(7)
    for f in (lambda p: L.nb200_dev_kv4_attention(p, P, 1 << 40, None), lambda p: L.nb200_dev_kv4_attention_workspace(p, C.byref(need))):
        refused(f(None), "null")
        refused(f(attention(head_dim=160, page_stride=8 * 40 * 160)), "no attention kernel")
        refused(f(attention(type=2)), "fp32 or bf16")
        refused(f(attention(heads=12)), "evenly")
        refused(f(attention(heads=0)), "evenly")
        refused(f(attention(batch=65536)), "65536 sequences")
        refused(f(attention(tokens=(1 << 30) + 1)), "too many")
        refused(f(attention(width=(1 << 25) + 1)), "too many")
        refused(f(attention(window=(1 << 30) + 1)), "2^30")
        refused(f(attention(softcap=-1.0)), "softcap")
        refused(f(attention(softcap=float("nan"))), "softcap")
        refused(f(attention(scale=float("inf"))), "scale")
        for name in ("q", "out", "lens", "table"):
            refused(f(attention(**{name: None})), "null")
        refused(f(attention(q=P + 1)), "aligned")
        refused(f(attention(out=P + 4)), "multiples of four")
        refused(f(attention(o_head=126)), "multiples of four")
        assert f(attention(batch=0)) == 0 and f(attention(tokens=0)) == 0
    refused(L.nb200_dev_kv4_attention_workspace(attention(), None), "null")


def test_a_cache_in_4_bits_is_refused_for_model_files():
    image, h = np.zeros(400, np.uint8), C.c_void_p()
    refused(E.lib().nb200_engine_create(C.byref(h), image.ctypes.data, image.size, 16, 0, E.FLAG_KV4), "model folders")
    assert not h.value


def test_waits_of_the_portion_kernel_end_for_a_warp_as_a_whole():
    """What a block of k_kv4_attn_tc does when a wait runs out is read from the source: whole warps get one verdict, two warps that meet at a barrier leave by what both know there, and it shows in
    their rows."""
    text = re.sub(r"//.*", "", open(os.path.join(ROOT, "nano_b200", "csrc", "kv4_tc.cu")).read())
    body = text[text.index("} else if (warp >= kMakers) {"):text.index("tc_dealloc")]
    makers, softmax = body.split("const uint32_t half = warp >> 2", 1)
    loop, end = softmax.split("sum_s[half][r] = l;", 1)
    waits = re.findall(r"(?:mbar_wait|soon)\w*\(", makers)
    assert len(waits) == 2 and set(waits) == {"soon_warp("} and len(re.findall(r"!soon_warp\([^;]*\)\) break;", makers)) == 2
    waits = re.findall(r"(?:mbar_wait|soon)\w*\(", loop)
    assert len(waits) == 4 and set(waits) == {"soon_warp("}, "a wait without one verdict for the warp"
    assert "__syncthreads" not in makers + loop and "bar.sync" not in body and loop.count("break;") == 1
    assert "if (!(ok = ok && ok_s[0][warp ^ 4u])) break;" in loop and "bar_any(id, 64u, !ok || top > m + kSlack)" in loop, "warps that part over a barrier"
    assert "ok = ok && ok_s[1][warp ^ 4u];" in end and "NAN;" in end and "if (n && ok) tc_ld16" in end
    one = text[text.index("auto scores = [&](uint32_t i)"):text.index("} else if (warp >= kMakers) {")]          # the thread that issues the products
    assert len(re.findall(r"soon\(", one)) == 4 and "soon_warp" not in one and "if (!ok) break;" in one and "i < n && ok" in one


@pytest.mark.skipif(E.device_count() > 0, reason="box has a GPU")
def test_no_cpu_fallback():
    L = E.lib()
    assert logprobs() == ENODEV
    assert pages([P], [0], [1]) == ENODEV
    assert L.nb200_dev_kv4_write(rows(), None) == ENODEV and L.nb200_dev_kv4_read(rows(), None) == ENODEV
    assert L.nb200_dev_kv4_attention(attention(), None, 0, None) == ENODEV
    from nano_b200 import ops
    import torch
    with pytest.raises(E.NB200Error, match="CUDA tensor"):
        ops.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(E.NB200Error, match="CUDA tensor"):
        ops.pages_copy([torch.zeros(4, 8)], [0], [1])
