"""Many completions of one prompt over the paged cache, against the same prompt
repeated through the contiguous cache (``models/decode.py``).

    python -m rs_nanogpt_b200.bench.samples [--samples 64] [--prompt 1500] [--new 128]

Random-init bf16 weights, random prompt, temperature 1, top-k 50, one GPU.
Reports the wall-clock milliseconds of a whole call (prompt upload to tokens on
the host, medians over ``--repeats``) and the key/value bytes that either holds.
"""
import argparse
import json
import random
import statistics
import time

import torch

from ..config import d_model
from ..models.decode import DecodeEngine, generate_batch
from ..models.paged import PagedDecoder
from ..models.params import ParamStore, init_params
from ..ops._ext import kernel_status


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--depth", type=int, default=20)
    p.add_argument("--vocab", type=int, default=65536)
    p.add_argument("--samples", type=int, default=64)
    p.add_argument("--prompt", type=int, default=1500)
    p.add_argument("--new", type=int, default=128)
    p.add_argument("--page", type=int, default=64)
    p.add_argument("--seed", type=int, default=0)
    p.add_argument("--repeats", type=int, default=3)
    a = p.parse_args(argv)
    dev = torch.device("cuda", 0)
    torch.cuda.set_device(dev)
    cfg = d_model(a.depth, vocab_size=a.vocab, sequence_len=2048)
    store = ParamStore(cfg, dev)
    init_params(store, seed=a.seed, mode="bench")
    store.refresh_work()
    rnd = random.Random(a.seed)
    prompt = [rnd.randrange(cfg.vocab_size) for _ in range(a.prompt)]
    length = a.prompt + a.new
    pages = a.prompt // a.page + a.samples * (-(-(a.prompt % a.page + a.new) // a.page))
    paged = PagedDecoder(store, pages, a.samples, length, a.page)
    engine = DecodeEngine(store, a.samples, -(-a.prompt // 256) * 256 + a.new)

    def timed(fn):
        fn()
        ms = []
        for _ in range(a.repeats):
            torch.cuda.synchronize()
            t = time.perf_counter()
            out = fn()
            torch.cuda.synchronize()
            ms.append((time.perf_counter() - t) * 1e3)
        assert len(out) == a.samples and all(len(o) == a.new for o in out)
        return statistics.median(ms)

    shared_ms = timed(lambda: paged.sample_many(prompt, a.samples, a.new, 1.0, 50, a.seed))
    repeated_ms = timed(lambda: generate_batch(engine, [prompt] * a.samples, a.new, 1.0, 50, a.seed))
    print(json.dumps({
        "metric": "completions of one prompt, random-init bf16", "shared_prefix_ms": shared_ms,
        "repeated_prompt_ms": repeated_ms, "samples": a.samples, "prompt_tokens": a.prompt, "new_tokens": a.new,
        "shared_prefix_kv_bytes": 2 * paged.cache.k.nbytes, "repeated_prompt_kv_bytes": 2 * engine.k_cache.nbytes,
        "kernel_status": kernel_status(), "config": {"model": f"GPT d{a.depth}", "vocab": cfg.vocab_size, "page": a.page},
    }))


if __name__ == "__main__":
    main()
