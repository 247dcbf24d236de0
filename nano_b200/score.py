"""Scores continuations of a prompt from the command line, for model folders and model files:

    python -m nano_b200.score --model DIR_OR_FILE --prompt-ids 5,17,3 --choice 9,4,11 --choice 9,7 [--top 3] [--dtype float32] [--cache 4bit]

Prints one JSON line per choice: the sum of the natural log probabilities of its tokens after the prompt, the log probability and the entropy at each of them and, with
--top, the most probable alternatives [id, log probability].  A model folder runs the prompt once and forks its sequence for every choice (Engine.seq_fork); the logits
stay on the device (Engine.step_scores, Engine.read_scores).
"""
from __future__ import annotations

import argparse
import json
import os
import sys


def _ids(text):
    return [int(x) for x in text.split(",") if x.strip()]


def score_folder(eng, prompt, choices, top):
    """(logprob, entropy, top_logprob, top_id) arrays of each choice's tokens, by forks of one sequence that holds the prompt."""
    seq = eng.seq_open()
    try:
        if len(prompt) > 1:
            eng.step(seq, prompt[:-1])
        for choice in choices:
            fork = eng.seq_fork(seq)
            try:
                yield eng.step_scores(fork, prompt[-1:] + choice[:-1], range(len(choice)), choice, top)
            finally:
                eng.seq_close(fork)
    finally:
        eng.seq_close(seq)


def score_file(eng, prompt, choices, top):
    """The same on the one implicit sequence of a model file, whose positions may be run again."""
    for pos, token in enumerate(prompt[:-1]):
        eng.forward_nolog(token, pos)
    for choice in choices:
        rows = []
        for i, (token, target) in enumerate(zip(prompt[-1:] + choice[:-1], choice)):
            eng.forward_nolog(token, len(prompt) - 1 + i)
            rows.append(eng.read_scores(target, top))
        yield tuple(zip(*rows))


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--model", required=True)
    ap.add_argument("--prompt-ids", required=True, help="comma-separated token ids")
    ap.add_argument("--choice", action="append", required=True, help="comma-separated token ids of one continuation; may be given many times")
    ap.add_argument("--top", type=int, default=0, help="alternatives to print at every token (at most 32)")
    ap.add_argument("--dtype", choices=["bfloat16", "float32"], default="bfloat16", help="model folders: compute type")
    ap.add_argument("--cache", choices=["32bit", "4bit"], default="32bit", help="model folders: how grouped-query attention layers hold keys and values")
    a = ap.parse_args(argv)
    prompt, choices = _ids(a.prompt_ids), [_ids(c) for c in a.choice]
    if not prompt or not all(choices):
        ap.error("the prompt and every choice need at least one token")
    from . import build as nb_build, engine as E
    folder = os.path.isdir(a.model)
    if folder and not os.path.exists(nb_build.ENGINE_SO):
        nb_build.build_layered()
    longest = max(len(c) for c in choices)
    room = len(prompt) + longest + (64 + longest if folder else 1)          # (a fork copies one page and adds its own tokens)
    eng = E.Engine(a.model, room, flags=(E.FLAG_F32 if (a.dtype == "float32" and folder) else 0) | (E.FLAG_KV4 if a.cache == "4bit" else 0))
    for choice, (lp, ent, tl, ti) in zip(choices, (score_folder if folder else score_file)(eng, prompt, choices, a.top)):
        row = {"choice": choice, "logprob": float(sum(float(x) for x in lp)), "token_logprobs": [float(x) for x in lp], "entropies": [float(x) for x in ent]}
        if a.top:
            row["top"] = [[[int(i), float(x)] for i, x in zip(ids, lps)] for ids, lps in zip(ti, tl)]
        print(json.dumps(row))
    eng.close()
    return 0


if __name__ == "__main__":
    sys.exit(main())
