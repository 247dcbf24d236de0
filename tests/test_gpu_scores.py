"""Scoring, forking and the cache in 4 bits through the engine: scores of wanted places against the logits that step() returns (in 64 bits), forks of a sequence against
sequences of their own in every registered design, grouped-query layers with a cache in 4 bits against the designs' oracles with rounded keys and values, and the command that
uses them together."""
import inspect
import json
import math
import os
import subprocess
import sys

import numpy as np
import pytest

from conftest import ROOT
from nano_b200 import engine as E, modeldir as md, modelfile as mf

import fidatar_oracle
import kadesun_oracle
import test_gpu_famudra
import test_gpu_fidatar
import test_gpu_gokinex
import test_gpu_kadesun
import test_gpu_rakarax
import test_gpu_vumunex

pytestmark = pytest.mark.gpu

MODULES = {"famudra": test_gpu_famudra, "rakarax": test_gpu_rakarax, "gokinex": test_gpu_gokinex, "vumunex": test_gpu_vumunex, "kadesun": test_gpu_kadesun, "fidatar": test_gpu_fidatar}
RANDOM = {n: getattr(md, n + "_random") for n in MODULES}


def build(tmp_path, cfg, design, flags=0, max_tokens=512, name="m", env=None):
    path = str(tmp_path / name)
    if not os.path.isdir(path):
        md.write_model_dir(path, cfg, RANDOM[design](cfg, 0))
    os.environ.update(env or {})
    try:
        return E.Engine(path, max_tokens, flags=flags)
    finally:
        for k in env or {}:
            os.environ.pop(k)


def toks(cfg, n, seed=1):
    return np.random.default_rng(seed).integers(0, cfg["vocab"], size=n).astype(np.uint32)


def check_scores(got, logits, targets, top):
    """log probabilities, entropies and alternatives of rows of fp32 logits: some dozens of roundings of 2^-24, and those of numbers as large as the logits"""
    lp, ent, tl, ti = got
    x = logits.astype(np.float64)
    peak = x.max(1, keepdims=True)
    z = np.exp(x - peak).sum(1, keepdims=True)
    want = x - peak - np.log(z)
    tol = 2.0 ** -24 * (128 + 8 * np.abs(want).max())
    assert np.abs(lp - want[np.arange(len(targets)), targets]).max() <= tol
    assert np.abs(ent + (np.exp(want) * want).sum(1)).max() <= tol * (1 + np.abs(ent).max())
    order = np.argsort(-logits, axis=1, kind="stable")[:, :top]
    assert np.array_equal(ti, order)
    if top:
        assert np.abs(tl - np.take_along_axis(want, order, 1)).max() <= tol


@pytest.mark.parametrize("design", list(MODULES))
@pytest.mark.parametrize("f32", [True, False])
def test_scores_of_steps(tmp_path, design, f32):
    cfg = MODULES[design].mixed_cfg()
    eng = build(tmp_path, cfg, design, E.FLAG_F32 if f32 else 0, env={"NB200_CHUNK": "96"})          # (portions of more tokens than a chunk holds, more places than one batch)
    t, goal = toks(cfg, 150), toks(cfg, 150, 2)
    a, b = eng.seq_open(), eng.seq_open()
    at = 0
    for n, want, top in [(110, range(0, 110), 5), (1, [0], 32), (2, [1], 0), (1, [], 3), (1, [0], 1), (30, [3, 4, 29], 7), (1, [0], 0), (4, [0, 3], 2)]:
        want = list(want)
        logits = eng.step(a, t[at:at + n], want)
        got = eng.step_scores(b, t[at:at + n], want, goal[at:at + n][want], top)
        assert got[0].shape == got[1].shape == (len(want),) and got[2].shape == got[3].shape == (len(want), top)
        if want:
            check_scores(got, logits, goal[at:at + n][want], top)
        at += n
    eng.step(b, t[:1])
    logits = eng.step(a, t[:1], [0])
    lp, ent, tl, ti = eng.read_scores(int(goal[0]), 4)
    check_scores((np.array([lp]), np.array([ent]), tl[None], ti[None]), logits, goal[:1], 4)
    eng.forward_nolog(int(t[0]), 0)          # the implicit sequence
    check_scores(tuple(np.asarray(x)[None] for x in eng.read_scores(3, 2)), eng.logits()[None], [3], 2)
    V = cfg["vocab"]
    for bad, text in [((b, t[:2], [1], [V], 0), "outside the vocabulary"), ((b, t[:2], [2], [0], 0), "ascending"), ((b, t[:2], [1, 0], [0, 0], 0), "ascending"), ((b, [V], [0], [0], 0), "outside the vocabulary"),
                      ((b, t[:2], [1], [0], 33), "at most 32"), ((7, t[:2], [1], [0], 0), "not open"), ((b, t[:2], [0, 1], [0], 0), "a target"), ((b, [], [], [], 0), "bad arguments")]:
        with pytest.raises(E.NB200Error, match=text):
            eng.step_scores(*bad)
    with pytest.raises(E.NB200Error, match="outside the vocabulary"):
        eng.read_scores(V)
    assert np.array_equal(eng.step(a, t[:3], [2]), eng.step(b, t[:3], [2]))          # a refused call has moved nothing
    eng.close()


@pytest.mark.parametrize("design", list(MODULES))
@pytest.mark.parametrize("length", [0, 1, 31, 32, 33, 77])
def test_forks_go_on_by_themselves(tmp_path, design, length):
    """Two forks and their source, continued in turn with tokens of their own, give the bits of sequences that never met."""
    cfg = MODULES[design].mixed_cfg()
    eng = build(tmp_path, cfg, design, max_tokens=900)
    pages = eng.free_pages
    prompt, tails = toks(cfg, length, 3), [toks(cfg, 70, 4 + i) for i in range(3)]
    cuts = [1, 1, 30, 3, 1, 34]

    def run(seqs, own):
        out = [[] for _ in own]
        at = 0
        for n in cuts:
            for i, s in enumerate(seqs):
                out[i].append(eng.step(s, own[i][at:at + n], range(n)))
            at += n
        return [np.concatenate(o) for o in out]
    alone = []
    for tail in tails:
        s = eng.seq_open()
        if length:
            eng.step(s, prompt)
        alone.append(run([s], [tail])[0])
        eng.seq_close(s)
    assert eng.free_pages == pages
    a = eng.seq_open()
    if length:
        eng.step(a, prompt)
    used = pages - eng.free_pages
    b = eng.seq_fork(a)
    c = eng.seq_fork(b)
    assert pages - eng.free_pages == used + (2 if length % 32 else 0)          # full pages are shared, the page in progress is copied
    for got, want in zip(run([a, b, c], tails), alone):
        assert np.array_equal(got, want)
    for s in (b, a, c):
        eng.seq_close(s)
    assert eng.free_pages == pages
    eng.close()


def test_forks_outlive_their_source_and_give_everything_back(tmp_path):
    cfg = test_gpu_fidatar.mixed_cfg()
    eng = build(tmp_path, cfg, "fidatar", max_tokens=512, env={"NB200_MAX_SEQS": "4"})
    pages, t = eng.free_pages, toks(cfg, 200)
    a = eng.seq_open()
    whole = eng.step(a, t[:120], range(120))
    b = eng.seq_fork(a)
    eng.seq_close(a)
    assert eng.free_pages == pages - 4
    other = eng.seq_open()          # the closed source's last page is written by another sequence
    eng.step(other, t[100:140])
    again = eng.seq_open()
    eng.step(again, t[:120])
    assert np.array_equal(eng.step(b, t[120:150], range(30)), eng.step(again, t[120:150], range(30)))
    c = eng.seq_fork(b)
    with pytest.raises(E.NB200Error, match="slots are in use"):
        eng.seq_fork(b)
    left = eng.free_pages
    eng.seq_close(c)
    assert eng.free_pages == left + 1          # (150 tokens: four pages shared, one its own)
    for bad in (c, 9):
        with pytest.raises(E.NB200Error, match="not open"):
            eng.seq_fork(bad)
    eng.seq_close(again)
    eng.step(other, toks(cfg, 32 * eng.free_pages))          # (fills the cache to its last page)
    while eng.free_pages:
        eng.step(other, t[:1])
    with pytest.raises(E.NB200Error, match="needs a page"):
        eng.seq_fork(b)
    s = eng.seq_open()          # the refused fork has left its slot free
    eng.seq_close(s)
    eng.seq_close(other)
    eng.seq_close(b)
    assert eng.free_pages == pages and whole.shape == (120, cfg["vocab"])
    eng.close()


@pytest.mark.parametrize("flags", [0, E.FLAG_NO_STREAM])
@pytest.mark.parametrize("name,quant", [("toy-nano", mf.QUANT_F32), ("toy-qwen3", mf.QUANT_Q80)])
def test_scores_of_model_files(name, quant, flags):
    spec = mf.PRESETS[name]
    eng = E.Engine(mf.cached_model(spec, quant, 64), 24, flags=flags)
    ids = np.zeros(25, np.uint32)
    ids[:6] = [3, 7, 1, 9, 4, 2]
    for pos in range(5):
        logits = eng.forward(int(ids[pos]), pos)
        check_scores(tuple(np.asarray(x)[None] for x in eng.read_scores(int(ids[pos + 1]), 6)), logits[None], ids[pos + 1:pos + 2], 6)
    eng.next_greedy(ids, 5, 0)
    check_scores(tuple(np.asarray(x)[None] for x in eng.read_scores(0, 1)), eng.logits()[None], [0], 1)
    with pytest.raises(E.NB200Error, match="outside the vocabulary"):
        eng.read_scores(spec.vocab)
    with pytest.raises(E.NB200Error, match="not available"):
        eng.seq_fork(0)
    eng.close()


# ---------------- the cache in 4 bits ----------------
def rounded(x):
    """rows [T, heads, D] as a cache in 4 bits holds them"""
    g = x.reshape(*x.shape[:-1], -1, 32)
    lo, hi = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
    m, s = lo.astype(np.float16).astype(np.float64), ((hi - lo) / 15).astype(np.float16).astype(np.float64)
    return (np.clip(np.round((g - m) / s), 0, 15) * s + m).reshape(x.shape)


def oracle4(module):
    """the module's forward() with keys and values rounded before they are attended to"""
    text = inspect.getsource(module.attention)
    mark = "    out = np.zeros((T, H, VD))"
    assert text.count(mark) == 1
    scope = dict(vars(module), rounded=rounded)
    exec(text.replace(mark, "    k, v = rounded(k), rounded(v)\n" + mark), scope)

    def forward(cfg, w, t):
        kept = module.attention
        module.attention = scope["attention"]
        try:
            return module.forward(cfg, w, t)
        finally:
            module.attention = kept
    return forward


def cfg4(design, dim, heads, kv_heads):
    if design == "fidatar":
        return md.fidatar_config(67, 56, [("attention", test_gpu_fidatar.att(dim=dim, vdim=dim, heads=heads, kv_heads=kv_heads, scale=dim ** -0.5), test_gpu_fidatar.dense(40)),
                                          ("mlstm", test_gpu_fidatar.MEM, None), ("attention", test_gpu_fidatar.att(dim=dim, vdim=dim, heads=heads, kv_heads=kv_heads, scale=dim ** -0.5, mask=None), None)], alpha=2.5)
    left = test_gpu_kadesun.left(dim=dim, vdim=dim, heads=heads, kv_heads=kv_heads, scale=dim ** -0.5)
    return md.kadesun_config(67, 56, [("parallel", test_gpu_kadesun.par(left), 40), ("delta", test_gpu_kadesun.DELTA, None), ("parallel", test_gpu_kadesun.par(left), None)])


@pytest.mark.parametrize("design,dim,heads,kv_heads", [("fidatar", 32, 6, 2), ("fidatar", 128, 4, 1), ("fidatar", 64, 3, 3), ("kadesun", 32, 6, 2), ("kadesun", 64, 8, 2), ("kadesun", 128, 2, 2)])
def test_layers_with_a_cache_in_4_bits(tmp_path, design, dim, heads, kv_heads):
    module, oracle = MODULES[design], {"fidatar": fidatar_oracle, "kadesun": kadesun_oracle}[design]
    cfg = cfg4(design, dim, heads, kv_heads)
    w = RANDOM[design](cfg, 0)
    t = toks(cfg, 190)
    exact, plain = oracle4(oracle)(cfg, w, t), oracle.forward(cfg, w, t)
    for n, (flags, cuts) in enumerate([(0, [190]), (0, [100] + [1] * 40 + [50]), (0, [33, 2, 3, 1, 64, 1, 1, 31, 4, 50]), (E.FLAG_NO_GRAPH | E.FLAG_NO_PDL, [120, 1, 1, 2, 66])]):
        eng = build(tmp_path, cfg, design, E.FLAG_KV4 | flags, env={"NB200_CHUNK": "80"} if n == 2 else None)
        got = module.in_cuts(eng, t, cuts)
        assert test_gpu_fidatar.close_bf16(got, exact)
        # it is the rounded rows that are attended to: nearer to their oracle than to the one of 32-bit rows
        assert np.median(module.rows(got, exact)) < 0.7 * np.median(module.rows(got, plain))
        eng.close()


def test_a_cache_in_4_bits_pages_forks_and_generation(tmp_path):
    cfg = cfg4("kadesun", 64, 8, 2)
    full, eng = build(tmp_path, cfg, "kadesun"), build(tmp_path, cfg, "kadesun", E.FLAG_KV4)
    t = toks(cfg, 150)
    a = eng.seq_open()
    eng.step(a, t[:75])
    b = eng.seq_fork(a)
    one = [eng.step(s, t[75:110], range(35)) for s in (a, b)]
    assert np.array_equal(*one)
    two = [eng.step(s, t[i:i + 1], [0]) for i in range(110, 120) for s in (a, b)]
    assert all(np.array_equal(x, y) for x, y in zip(two[::2], two[1::2]))
    got = eng.step_scores(b, t[120:140], range(20), t[121:141], 2)
    check_scores(got, eng.step(a, t[120:140], range(20)), t[121:141], 2)
    assert eng.step_timed(a, t[:10], 2) > 0
    eng.seq_close(a), eng.seq_close(b)
    ids = np.zeros(61, np.uint32)
    ids[:20] = t[:20]
    eng.decode_greedy(ids, 20, 60)
    s = eng.seq_open()
    logits = eng.step(s, ids[:59], range(59))
    # the tokens chosen one by one are the largest logits of the whole (or as large but for the rounding of bfloat16 products)
    chosen = logits[np.arange(19, 59), ids[20:60]]
    assert (chosen >= logits[19:59].max(1) - 0.05 * np.abs(logits).max()).all()
    full.close(), eng.close()


def _lp(x):
    x = x.astype(np.float64)
    return x - x.max(1, keepdims=True) - np.log(np.exp(x - x.max(1, keepdims=True)).sum(1, keepdims=True))


def test_a_long_cache_in_4_bits(tmp_path):
    """Contexts whose keys are split over blocks, in captured steps too, against portions of the same tokens."""
    cfg = md.fidatar_config(67, 64, [("attention", test_gpu_fidatar.att(dim=64, vdim=64, heads=8, kv_heads=2, scale=0.125, mask=None, rot=None), None)], alpha=2.5)
    eng = build(tmp_path, cfg, "fidatar", E.FLAG_KV4, max_tokens=9000)
    t = toks(cfg, 4100)
    a, b = eng.seq_open(), eng.seq_open()
    eng.step(a, t[:4000]), eng.step(b, t[:4000])
    one = np.concatenate([eng.step(a, t[i:i + 1], [0]) for i in range(4000, 4030)])
    many = eng.step(b, t[4000:4030], range(30))
    d = one - many
    assert np.sqrt((d ** 2).mean()) < 2e-2 * np.sqrt((many ** 2).mean())
    eng.close()


def test_a_cache_in_4_bits_is_refused_where_there_is_none(tmp_path):
    for design, cfg, flags, text in [("famudra", test_gpu_famudra.mixed_cfg(), 0, "no grouped-query"), ("fidatar", test_gpu_fidatar.mixed_cfg(), 0, "dim 20 and vdim 12"), ("fidatar", cfg4("fidatar", 32, 2, 1), E.FLAG_F32, "exclude each other"),
                                     ("kadesun", md.kadesun_config(67, 56, [("parallel", test_gpu_kadesun.par(test_gpu_kadesun.left(dim=32, vdim=64)), None)]), 0, "dim 32 and vdim 64")]:
        with pytest.raises(E.NB200Error, match=text):
            build(tmp_path, cfg, design, E.FLAG_KV4 | flags, name=f"{design}{text[:6].strip()}")


# ---------------- the command ----------------
@pytest.mark.parametrize("cache", ["32bit", "4bit"])
def test_score_command(tmp_path, cache):
    cfg = cfg4("fidatar", 32, 2, 1)
    path = str(tmp_path / "m")
    md.write_model_dir(path, cfg, RANDOM["fidatar"](cfg, 0))
    prompt, choices = toks(cfg, 45).tolist(), [toks(cfg, n, 5 + n).tolist() for n in (1, 4, 40)]
    out = subprocess.run([sys.executable, "-m", "nano_b200.score", "--model", path, "--prompt-ids", ",".join(map(str, prompt)), "--top", "3", "--cache", cache] +
                         [a for c in choices for a in ("--choice", ",".join(map(str, c)))], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    lines = [json.loads(x) for x in out.stdout.splitlines()]
    assert [x["choice"] for x in lines] == choices
    eng = E.Engine(path, 256, flags=E.FLAG_KV4 if cache == "4bit" else 0)
    for c, line in zip(choices, lines):
        s = eng.seq_open()
        eng.step(s, prompt[:-1])
        lp = _lp(eng.step(s, prompt[-1:] + c[:-1], range(len(c))))
        eng.seq_close(s)
        want = lp[np.arange(len(c)), c]
        assert np.abs(np.array(line["token_logprobs"]) - want).max() < 1e-4 and math.isclose(line["logprob"], want.sum(), abs_tol=1e-3)
        assert [[i for i, _ in row] for row in line["top"]] == np.argsort(-lp, 1, kind="stable")[:, :3].tolist()
    eng.close()


def test_score_command_of_a_model_file():
    spec = mf.PRESETS["toy-qwen3"]
    path = mf.cached_model(spec, mf.QUANT_Q80, 64)
    out = subprocess.run([sys.executable, "-m", "nano_b200.score", "--model", path, "--prompt-ids", "11,22,33", "--choice", "4,5", "--choice", "6"], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    lines = [json.loads(x) for x in out.stdout.splitlines()]
    eng = E.Engine(path, 8)
    for pos, token in enumerate((11, 22, 33, 4)):
        lp = _lp(eng.forward(token, pos)[None])[0]
        if pos >= 2:
            assert abs(lines[0]["token_logprobs"][pos - 2] - lp[(4, 5)[pos - 2]]) < 1e-4
        if pos == 2:
            assert abs(lines[1]["logprob"] - lp[6]) < 1e-4
    eng.close()
