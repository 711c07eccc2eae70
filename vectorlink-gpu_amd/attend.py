"""Command line example: a few sequences are read in and answered over a key/value cache held in 4 bits.

    python vectorlink-gpu_amd/attend.py -c 32768 -b 4 -k 32

Keys and values are random around a subject for every 256 tokens, and every new token asks about one of the subjects.  The
context is read in pieces (write, attend); then every step writes a token of each sequence and attends once to everything
and once to the `-k` blocks that its 8-bit bounds choose.  Prints what a step takes both ways, how far the choice is from
everything, and how far 4 bits are from the numbers that were written, as JSON.
"""
import argparse
import json
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

# (short flag, long flag, default, help) for the integer options
INT_OPTIONS = [
    ("-c", "--context", 32_768, "tokens read in before the answer"),
    ("-b", "--sequences", 4, "sequences answered at once"),
    ("-n", "--heads", 8, "heads of the cache"),
    ("-g", "--group", 4, "heads of queries that share one"),
    ("-d", "--dimension", 128, "dimensions of a head"),
    ("-k", "--count", 32, "blocks of 64 tokens that a token chooses"),
    ("-p", "--piece", 2_048, "tokens of a sequence that are read in at once"),
    ("-s", "--steps", 64, "tokens of the answer"),
]


def at_least_one(text: str) -> int:
    n = int(text)
    if n < 1:
        raise argparse.ArgumentTypeError(f"at least 1, got {n}")
    return n


def parse(argv=None) -> dict:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for short, long_, default, text in INT_OPTIONS:
        parser.add_argument(short, long_, type=at_least_one, default=default, help=text)
    return vars(parser.parse_args(argv))


def main(options: dict, seed: int = 0) -> dict:
    import torch

    from vectorlink_gpu.attention import PAGE, KVCache, attend, attend_selected

    (context, batch, heads, group, dim) = (options[k] for k in ("context", "sequences", "heads", "group", "dimension"))
    (count, piece, steps) = (options[k] for k in ("count", "piece", "steps"))
    device = "cuda"
    gen = torch.Generator(device=device).manual_seed(seed)
    blocks = -(-(context + steps) // PAGE)
    cache = KVCache.empty(batch * blocks, heads, dim, device=device)
    table = torch.randperm(batch * blocks, generator=gen, device=device).to(torch.int32).view(batch, blocks)
    lengths = torch.zeros(batch, dtype=torch.int32, device=device)
    subjects = torch.randn((batch, -(-(context + steps) // 256), heads, dim), generator=gen, device=device)

    def tokens(first: int, n: int):
        """Queries, keys and values [batch * n, heads, dim] of n tokens of every sequence, side by side as one projection gives them."""
        mixed = torch.randn((batch, n, heads * (group + 2), dim), generator=gen, device=device)
        about = torch.arange(first, first + n, device=device) // 256
        mixed[:, :, heads * group:heads * (group + 1)] += subjects[:, about]
        asked = torch.randint(0, max(1, context // 256), (n,), generator=gen, device=device)
        mixed[:, :, :heads * group] += subjects[:, asked].repeat_interleave(group, dim=2)
        mixed = mixed.flatten(0, 1).bfloat16()
        return mixed[:, :heads * group], mixed[:, heads * group:heads * (group + 1)], mixed[:, heads * (group + 1):]

    def clock() -> float:
        torch.cuda.synchronize()
        return time.perf_counter()

    read_in, written, seen = 0.0, [], 0
    while seen < context:
        n = min(piece, context - seen)
        (q, k, v) = tokens(seen, n)
        offsets = torch.arange(0, batch * n + 1, n, dtype=torch.int32, device=device)
        began = clock()
        cache.write(k, v, table, lengths, offsets)
        lengths += n
        attend(q, cache, table, lengths, offsets)
        read_in += clock() - began
        written.append((k, v))
        seen += n
    # what 4 bits leave of the last piece, as a share of its length
    (k4, v4) = cache.read(table, lengths - n, batch * n, offsets)
    far = [float((a.float() - b.float()).norm() / b.float().norm()) for a, b in zip((k4, v4), written[-1])]

    took = {"all": 0.0, "chosen": 0.0}
    off = []
    for step in range(steps):
        (q, k, v) = tokens(context + step, 1)
        cache.write(k, v, table, lengths)
        lengths += 1
        began = clock()
        whole = attend(q, cache, table, lengths)
        between = clock()
        (chosen, ids) = attend_selected(q, cache, table, lengths, count)
        if step:  # the first step loads the kernels
            took["all"] += between - began
            took["chosen"] += clock() - between
        off.append(float((chosen.float() - whole.float()).norm() / whole.float().norm()))
    report = dict(options)
    report.update(read_in_ms=1e3 * read_in, step_all_us=1e6 * took["all"] / max(1, steps - 1), step_chosen_us=1e6 * took["chosen"] / max(1, steps - 1),
                  chosen_off=sum(off) / len(off), keys_off=far[0], values_off=far[1],
                  bytes_a_token=heads * (dim + dim // 16), blocks=blocks)
    return report


if __name__ == "__main__":
    print(json.dumps(main(parse())))
