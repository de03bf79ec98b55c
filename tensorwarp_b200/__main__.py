"""Command line: ``python -m tensorwarp_b200 generate|trace|models``."""
from __future__ import annotations

import argparse
import json
import sys


def _generate(args) -> int:
    import torch

    from . import registry
    from .scheduler import Scheduler
    options = {"max_live": args.max_live}
    if args.max_tokens:
        options["max_tokens"] = args.max_tokens
    if args.kv_cache:
        options["kv_cache"] = args.kv_cache
    sampling = None
    if args.temperature is None and (args.top_k, args.top_p, args.min_p) != (0, 1.0, 0.0):
        raise SystemExit("generate: --top-k, --top-p and --min-p want a --temperature")
    if args.temperature is not None:
        from .sampling import SamplingParams
        sampling = [SamplingParams(args.temperature, args.top_k, args.top_p, args.min_p, args.seed + i) for i in range(len(args.tokens))]
    engine = registry.load(args.model, dtype={"bfloat16": torch.bfloat16, "float32": torch.float32}[args.dtype], **options)
    scheduler = Scheduler(engine, portion=args.portion)
    index = {}
    for i, text in enumerate(args.tokens):
        request = scheduler.submit([int(t) for t in text.split(",")], args.max_new_tokens, args.stop_token, sampling[i] if sampling else None)
        index[id(request)] = i
    for request in scheduler.run():
        print(json.dumps({"request": index[id(request)], "generated": request.generated}), flush=True)
    return 0


def _models(args) -> int:
    from . import registry
    print("\n".join(registry.architectures()))
    return 0


def _trace(args) -> int:
    from . import trace
    return trace.main(args)


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(prog="tensorwarp_b200")
    sub = ap.add_subparsers(dest="command", required=True)
    g = sub.add_parser("generate", help="generation from token ids, greedily or sampled")
    g.add_argument("--model", required=True, help="folder with config.json and model.safetensors")
    g.add_argument("--tokens", required=True, action="append", help="a prompt as comma-separated token ids (repeat for more)")
    g.add_argument("--max-new-tokens", type=int, default=16)
    g.add_argument("--stop-token", type=int, default=None)
    g.add_argument("--dtype", choices=["bfloat16", "float32"], default="bfloat16")
    g.add_argument("--max-tokens", type=int, default=None, help="longest sequence to make room for")
    g.add_argument("--max-live", type=int, default=4, help="sequences in flight at once")
    g.add_argument("--portion", type=int, default=2048, help="most prompt tokens per step")
    g.add_argument("--temperature", type=float, default=None, help="sample at this temperature (without it: greedily)")
    g.add_argument("--top-k", type=int, default=0, help="sample among this many tokens (0: all)")
    g.add_argument("--top-p", type=float, default=1.0, help="... among the likeliest that hold this share")
    g.add_argument("--min-p", type=float, default=0.0, help="... among those at least this likely beside the likeliest")
    g.add_argument("--seed", type=int, default=0, help="of the first prompt's random numbers; the next one's is one more")
    g.add_argument("--kv-cache", choices=["f16", "e4m3"], default=None, help="how the 4-bit decoder holds keys and values")
    g.set_defaults(run=_generate)
    t = sub.add_parser("trace", help="replay a trace of steps from standard input and write the logits it asks for")
    t.add_argument("--model", required=True)
    t.add_argument("--dtype", choices=["bfloat16", "float32"], required=True)
    t.add_argument("--out", required=True, help="folder for <step>.f32")
    t.add_argument("--max-tokens", type=int, required=True, help="room for this many tokens per sequence")
    t.set_defaults(run=_trace)
    m = sub.add_parser("models", help="list the architectures")
    m.set_defaults(run=_models)
    args = ap.parse_args(argv)
    return args.run(args)


if __name__ == "__main__":
    sys.exit(main())
