"""Whole decoding steps of a beam search, at the sizes of the models bench.py runs (random weights, bfloat16, pages of 16).

    python perf/beam_steps.py [--models 135M,360M,1.7B] [--beams 8,64] [--prompts 2000,8000] [--ctx 8192]

A line for each model, number of beams and prompt, milliseconds a step: the search as the engine's rule runs it, the search with common pages read once, with every beam's
pages read by themselves; and the model's steps alone, issued one after the other without a choice between them, both ways.  Of a search the difference of one of
`--steps` + 2 tokens and one of 2, the least of three.
"""
import argparse
import os
import sys
import tempfile
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from perf.cases import LLAMA  # noqa: E402
from vitna_anchor_b200 import ops  # noqa: E402
from vitna_anchor_b200.engine.engine import Engine  # noqa: E402
from vitna_anchor_b200.engine.loading import write_random_model  # noqa: E402
from vitna_anchor_b200.engine.runner import StepEntry  # noqa: E402

PAGE = 16


def config(c):
    return dict(architectures=["LlamaForCausalLM"], model_type="llama", hidden_act="silu", num_hidden_layers=c["layers"], hidden_size=c["hidden"], intermediate_size=c["inter"],
                num_attention_heads=c["heads"], num_key_value_heads=c["kv"], head_dim=c["dim"], vocab_size=c["vocab"], max_position_embeddings=131072, rms_norm_eps=1e-5,
                rope_theta=c["theta"], tie_word_embeddings=True)


def seconds(fn):
    torch.cuda.synchronize()
    t = time.perf_counter()
    fn()
    torch.cuda.synchronize()
    return time.perf_counter() - t


def search_ms(eng, prompt, beams, mode, steps):
    ops.set_attention_shared(mode)
    for n in (steps + 2, 2, steps + 2):
        eng.beam_search(prompt, beams=beams, max_new=n)
    best = min(seconds(lambda: eng.beam_search(prompt, beams=beams, max_new=steps + 2)) - seconds(lambda: eng.beam_search(prompt, beams=beams, max_new=2)) for _ in range(3))
    ops.set_attention_shared(2)
    return best / steps * 1e3


def alone_ms(eng, prompt, beams, mode, steps):
    ops.set_attention_shared(mode)
    r, least = eng.runner, float("inf")
    for _ in range(4):
        r.open("b0")
        for at in range(0, len(prompt), r.max_batch_tokens):
            r.step([StepEntry("b0", prompt[at:at + r.max_batch_tokens], [])])
        r.fork_many([(f"b{i}", "b0") for i in range(1, beams)])
        entries = [StepEntry(f"b{i}", [7 + i], [0]) for i in range(beams)]
        r.step(entries)
        least = min(least, seconds(lambda: [r.step(entries) for _ in range(steps)]))
        r.check()
        for i in range(beams):
            r.close(f"b{i}")
    ops.set_attention_shared(2)
    return least / steps * 1e3


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--models", default="135M,360M,1.7B")
    ap.add_argument("--beams", default="8,64")
    ap.add_argument("--prompts", default="2000,8000")
    ap.add_argument("--ctx", type=int, default=8192)
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args()
    for name in a.models.split(","):
        c = LLAMA[name]
        with tempfile.TemporaryDirectory() as folder:
            write_random_model(folder, config(c), 0)
            for beams in map(int, a.beams.split(",")):
                for length in map(int, a.prompts.split(",")):
                    eng = Engine(folder, dtype="bfloat16", ctx=a.ctx, parallel=beams, num_pages=length // PAGE + beams * (a.steps // PAGE + 3) + 8)
                    prompt = torch.randint(0, c["vocab"], (length,), generator=torch.Generator().manual_seed(length)).tolist()
                    rule, once, apart = (search_ms(eng, prompt, beams, mode, a.steps) for mode in (2, 1, 0))
                    alone = [alone_ms(eng, prompt, beams, mode, a.steps) for mode in (1, 0)]
                    saved = (beams - 1) * length * c["kv"] * c["dim"] * 4 / 2 ** 20
                    print(f"{name:5s} {beams:3d} beams of {length:6d} ({saved:6.0f} MB read again a layer): search {rule:7.3f}, once {once:7.3f}, apart {apart:7.3f}; steps alone "
                          f"once {alone[0]:7.3f}, apart {alone[1]:7.3f}", flush=True)
                    del eng
                    torch.cuda.empty_cache()


if __name__ == "__main__":
    main()
