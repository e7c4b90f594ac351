"""Command line:

    python -m baranet_bdml_b200 generate --model DIR [--dtype bfloat16] [--max-new-tokens N] [--temperature T] [--top-k K] [--top-p P]
        [--min-p R] [--seed S] [--kv-cache bf16] --prompt "5 17 3" [--prompt ...]
    python -m baranet_bdml_b200 trace --model DIR --out DIR < steps.jsonl

`generate` continues prompts of token ids and prints one line of ids per prompt: greedily, or sampled with a temperature above 0."""
from __future__ import annotations

import argparse
import sys


def generate(argv) -> int:
    ap = argparse.ArgumentParser(prog="generate")
    ap.add_argument("--model", required=True, help="folder with config.json and model.safetensors")
    ap.add_argument("--dtype", default="bfloat16", choices=["bfloat16", "float32"])
    ap.add_argument("--max-new-tokens", type=int, default=50)
    ap.add_argument("--prompt", action="append", required=True, help="token ids, separated by spaces or commas")
    ap.add_argument("--temperature", type=float, default=0.0, help="0: the likeliest id")
    ap.add_argument("--top-k", type=int, default=0, help="of the likeliest K ids (0: all)")
    ap.add_argument("--top-p", type=float, default=1.0, help="of those that have this much of the probability together")
    ap.add_argument("--min-p", type=float, default=0.0, help="of those with at least this share of the likeliest one's probability")
    ap.add_argument("--seed", type=int, default=None, help="the same seed gives the same ids")
    ap.add_argument("--kv-cache", default="bf16", choices=["bf16", "e4m3", "int8"], help="what the LLaMA model's cache holds")
    a = ap.parse_args(argv)
    from . import registry
    prompts = [[int(t) for t in p.replace(",", " ").split()] for p in a.prompt]
    model = registry.load_model(a.model, a.dtype)
    if a.kv_cache != "bf16":
        if not hasattr(model, "kv_cache"):
            ap.error("--kv-cache: this model's cache is of its own kind")
        model.kv_cache = a.kv_cache
    for row in model.generate(prompts, a.max_new_tokens, temperature=a.temperature, top_k=a.top_k, top_p=a.top_p, min_p=a.min_p, seed=a.seed):
        print(*row)
    model.status()
    return 0


def main(argv=None) -> int:
    argv = list(sys.argv[1:] if argv is None else argv)
    if argv[:1] == ["generate"]:
        return generate(argv[1:])
    if argv[:1] == ["trace"]:
        from .trace import main as trace
        return trace(argv[1:])
    print(__doc__, file=sys.stderr)
    return 2


if __name__ == "__main__":
    sys.exit(main())
