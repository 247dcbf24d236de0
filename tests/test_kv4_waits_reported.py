"""A wait that runs out in the attention of portions over a cache in 4 bits reaches the caller of the engine as an error, not as NaN alone.  That is not run (it would take a broken kernel) but read
from the source: the kernel's rows become NaN and its error word is set by one verdict, the engine hands its word over, and every step looks at it once the device is done."""
import os
import re

from conftest import ROOT


def source(name):
    return re.sub(r"//.*", "", open(os.path.join(ROOT, "nano_b200", "csrc", name)).read())


def test_the_kernel_sets_the_word_where_its_rows_are_lost():
    text = source("kv4_tc.cu")
    end = text[text.index("sum_s[half][r] = l;"):text.index("tc_dealloc")]
    verdict, word, rows = (end.index(x) for x in ("ok = ok && ok_s[1][warp ^ 4u];", "if (!ok && lane == 0 && a.err) *a.err = ", "sum = ok ? l + sum_s[half ^ 1u][r] : NAN"))
    assert verdict < word < rows and not re.search(r"\bok = ", end[verdict + 5:])


def test_the_engine_hands_its_word_over_and_looks_at_it():
    text = source("layered.cu")
    branch = text[text.index("nb::Kv4Attn ka{}"):text.index("nb::kv4_attn_launch(")]
    assert "ka.err = e->tc.err_dev;" in branch
    assert re.search(r"if \(e->kv4 && \(r = tc_error_word\(&e->tc\)\)\) return r;", text)
    step = text[text.index("int step_any("):text.index("int lm_step(")]
    ends = re.findall(r"return (?:0|fetch_logits\([^;]*|score_rows\([^;]*|tc_check\(&e->tc\));", step)
    assert ends == ["return tc_check(&e->tc);"] * 3, ends
    for name in ("lm_step_timed", "lm_forward", "lm_next_greedy", "lm_next_sampled", "lm_decode_greedy"):
        body = text[text.index("int %s(" % name):]
        assert body[:body.index("\n}\n")].rstrip().endswith("return tc_check(&e->tc);"), name
