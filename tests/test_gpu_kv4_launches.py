"""How the kernels of the cache in 4 bits follow one another: an engine that was told not to launch a kernel while the one before it runs (NB200_FLAG_NO_PDL) launches none of them so, the join of a
row's splits among them, and computes the same bits."""
import os
import re

import numpy as np
import pytest

from conftest import ROOT
from nano_b200 import engine as E, modeldir as md


def test_who_says_so():
    text = re.sub(r"//.*", "", open(os.path.join(ROOT, "nano_b200", "csrc", "kv4.cu")).read())
    launches = re.findall(r"launch_on\((k_kv4_\w+).*?, stream, (\w+), a", text)
    assert ("k_kv4_join", "pdl_join") in launches and "true" not in [x[1] for x in launches], launches
    engine = open(os.path.join(ROOT, "nano_b200", "csrc", "layered.cu")).read()
    assert "nb::kv4_attn_launch(ka, (uint32_t)e->num_sms, e->cur, e->use_pdl, e->use_pdl, &launches)" in engine


@pytest.mark.gpu
def test_an_engine_without_pdl(tmp_path):
    import test_gpu_fidatar
    from test_gpu_scores import build, toks
    cfg = md.fidatar_config(67, 64, [("attention", test_gpu_fidatar.att(dim=64, vdim=64, heads=8, kv_heads=2, scale=0.125, mask=None, rot=None), None)], alpha=2.5)
    got = []
    for flags in (E.FLAG_KV4, E.FLAG_KV4 | E.FLAG_NO_PDL):
        eng = build(tmp_path, cfg, "fidatar", flags, max_tokens=4200)
        s = eng.seq_open()
        eng.step(s, toks(cfg, 4000))          # (single tokens behind 4000: their keys are split)
        got.append(np.concatenate([eng.step(s, toks(cfg, n, n), range(n)) for n in (1, 1, 5, 40)]))
        eng.close()
    assert np.isfinite(got[0]).all() and np.array_equal(got[0].view(np.uint32), got[1].view(np.uint32))
