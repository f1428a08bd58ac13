"""Greedy generation from the command line:

    python -m nn_b200.generate --model PATH --prompt 11,4,90 --new 32 [--dtype bfloat16|float32] [--max-seq N]
                               [--cache f32|int8|e4m3] [--logprobs K]

PATH is a model folder (config.json + model.safetensors) or a GGUF file; prompt and output are token ids. --cache keeps the keys
and values of a Qwen3 model in 8 bits. With --logprobs nothing is generated: a line for each token of the prompt behind the first with its log
probability, the entropy in its place and the K most probable tokens there.
"""
from __future__ import annotations

import argparse
import sys

from . import kv_cache, models
from .trace import DTYPES


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(prog="python -m nn_b200.generate", description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--model", required=True)
    ap.add_argument("--prompt", required=True, help="token ids with commas between them")
    ap.add_argument("--new", type=int, default=16, help="tokens to generate")
    ap.add_argument("--dtype", default="bfloat16", choices=sorted(DTYPES))
    ap.add_argument("--max-seq", type=int, default=0, help="positions held (default: prompt + new)")
    ap.add_argument("--cache", default="f32", choices=["f32", "int8", "e4m3"], help="keys and values of a Qwen3 model")
    ap.add_argument("--logprobs", type=int, default=None, metavar="K", help="score the prompt instead")
    a = ap.parse_args(argv)
    prompt = [int(t) for t in a.prompt.split(",")]
    dec = models.load_model(a.model, max_seq=a.max_seq or len(prompt) + a.new, act_dtype=DTYPES[a.dtype])
    if a.cache != "f32":
        dec.set_cache({"int8": kv_cache.INT8, "e4m3": kv_cache.E4M3}[a.cache])
    if a.logprobs is not None:
        r = dec.score(prompt, top=a.logprobs)
        for i, t in enumerate(prompt[1:]):
            best = "" if r.top_tokens is None else "  " + " ".join(f"{k}:{p:.4f}" for k, p in zip(r.top_tokens[i].tolist(), r.top_logprobs[i].tolist()))
            print(f"{t} {r.logprob[i]:.4f} {r.entropy[i]:.4f}{best}")
        return 0
    print(",".join(str(t) for t in dec.complete(prompt, a.new)))
    return 0


if __name__ == "__main__":
    sys.exit(main())
