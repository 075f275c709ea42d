"""A prompt's keys and values in a 4-bit cache laid out by k-means, and decoding steps that look at a few of its pages.

  python examples/cache4_decode.py [--prompt 16384] [--steps 32] [--heads 4] [--group 4] [--dim 128] [--page 64] [--pages 24]

1. k-means in one dimension learns the 8 levels of each head's quantiser from a sample of the rows (cache4_learn_levels).
2. k-means in `dim` dimensions clusters the prompt's keys; the rows go to the cache cluster by cluster, so that a page holds keys that are alike and
   its bounds are tight. (Attention does not ask for the order of the tokens it sees; positions are in the keys.)
3. Each step writes its token behind the prompt, refreshes the bounds of that page, chooses pages by their scores and attends to them.
The last step is compared with attention to the whole cache and with that to the unquantised rows, the layout with that of the prompt's own order.
"""
import argparse
import importlib
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
km = importlib.import_module("cuda-kmeans_amd")


def bf16(x):
    """float32 values rounded to bfloat16, as stored."""
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
    return ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def floats(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def device(array):
    a = np.ascontiguousarray(array)
    buffer = km.DeviceBuffer(a.nbytes)
    buffer.write(a)
    return buffer


def order_by_clusters(keys, page):
    """The prompt's tokens cluster by cluster: k-means on the keys of all heads side by side, about a cluster a page."""
    n = keys.shape[0]
    rows = np.ascontiguousarray(keys.reshape(n, -1))
    k = max(1, n // page)
    alg = km.HipKMeansAlgorithm()
    alg.initialize(rows.shape[1], k, n, 8, rows.reshape(-1), rows[np.linspace(0, n - 1, k).astype(int)].reshape(-1))
    alg.run()
    cluster = alg.getAssignment()
    alg.cleanup()
    return np.argsort(cluster, kind="stable")


def run(prompt=16384, steps=32, heads=4, group=4, dim=128, page=64, pages=24, seed=0, say=print):
    rng = np.random.default_rng(seed)
    topics = rng.normal(size=(96, heads, dim)) * 1.5
    topic = rng.integers(0, 96, prompt + steps)
    keys = floats(bf16(topics[topic] + 0.6 * rng.normal(size=(prompt + steps, heads, dim))))
    values = floats(bf16(rng.normal(size=(prompt + steps, heads, dim))))
    queries = floats(bf16(0.3 * topics[topic[prompt:]][:, :, None] + 0.5 * rng.normal(size=(steps, heads, group, dim))))
    scale = 1 / np.sqrt(dim)

    sample = rng.permutation(prompt)[:4096]
    levels = np.stack([np.stack([km.cache4_learn_levels(x[sample, h]) for x in (keys, values)]) for h in range(heads)])
    count = -(-(prompt + steps) // page)
    block_bytes, bound_bytes = km.Cache4.sizes(heads, dim, page, count)
    say("cache: %d tokens in %d pages, %.1f MB (rows in bf16: %.1f MB), bounds %.2f MB" % (prompt + steps, count, block_bytes / 1e6, 4e-6 * (prompt + steps) * heads * dim, bound_bytes / 1e6))
    result = {}
    for name, order in (("prompt's order", np.arange(prompt)), ("by clusters", order_by_clusters(keys[:prompt], page))):
        cache = km.Cache4(heads, dim, page, count, device(levels), km.DeviceBuffer(block_bytes), km.DeviceBuffer(bound_bytes))
        cache.write(km.TYPE_BF16, device(bf16(keys[order])), device(bf16(values[order])), device(np.arange(prompt, dtype=np.int32)), prompt)
        full = prompt // page
        used = -(-prompt // page)
        counts = np.full(used, page, np.int32)
        counts[full:] = prompt % page
        cache.bound(device(np.arange(used, dtype=np.int32)), device(counts), used)
        q, k, v = device(bf16(queries)), device(bf16(keys[prompt:])), device(bf16(values[prompt:]))
        table = device(np.arange(count, dtype=np.int32))
        out, whole = km.DeviceBuffer(2 * heads * group * dim), km.DeviceBuffer(2 * heads * group * dim)
        chosen = km.DeviceBuffer(4 * heads * pages)
        small = device(np.arange(prompt, prompt + steps, dtype=np.int32))          # places of the steps' tokens
        page_of = device(np.arange(prompt, prompt + steps, dtype=np.int32) // page)  # their pages, and how many tokens those hold then
        filled = device(np.arange(prompt, prompt + steps, dtype=np.int32) % page + 1)
        starts, lengths = device(np.int32([0, 1])), device(np.arange(prompt + 1, prompt + steps + 1, dtype=np.int32))
        part = lambda buffer, at, size: km.DeviceView(buffer.ptr.value + at * size, size)  # noqa: E731
        batch = [km.Cache4Batch(1, heads * group, 1, 1, prompt + steps, starts, part(lengths, i, 4), table, count) for i in range(steps)]
        cache.reserve(batch[0], pages)
        begin, end = km.Event(), km.Event()
        for i in [0] + list(range(steps)):  # the first step twice: once to warm up
            if i == 0:
                begin.record()
            row, query = 2 * heads * dim, part(q, i, 2 * heads * group * dim)
            cache.write(km.TYPE_BF16, part(k, i, row), part(v, i, row), part(small, i, 4), 1)
            cache.bound(part(page_of, i, 4), part(filled, i, 4), 1)
            cache.select(batch[i], km.TYPE_BF16, query, chosen, pages)
            cache.attend(batch[i], km.TYPE_BF16, query, out, scale, chosen=chosen, top=pages)
        end.record()
        km.sync()
        took = begin.elapsed_ms(end) / steps * 1e3
        cache.attend(batch[-1], km.TYPE_BF16, query, whole, scale)
        km.sync()
        got, all_pages = (floats(b.read(np.uint16, heads * group * dim)).reshape(heads, group, dim).astype(np.float64) for b in (out, whole))
        score = scale * np.einsum("hgd,thd->hgt", queries[-1].astype(np.float64), keys.astype(np.float64))
        p = np.exp(score - score.max(-1, keepdims=True))
        exact = np.einsum("hgt,thd->hgd", p / p.sum(-1, keepdims=True), values.astype(np.float64))
        off = lambda x: float(np.linalg.norm(x - exact) / np.linalg.norm(exact))  # noqa: E731
        result[name] = dict(us=took, sparse=off(got), whole=off(all_pages))
        say("%-15s %6.1f us a step with %d of %d pages; the last step's output is off by %.3f, with all pages by %.3f" % (name + ":", took, pages, count, off(got), off(all_pages)))
    return result


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for option, value in (("prompt", 16384), ("steps", 32), ("heads", 4), ("group", 4), ("dim", 128), ("page", 64), ("pages", 24), ("seed", 0)):
        parser.add_argument("--" + option, type=int, default=value)
    km.check(km.hip_lib().kmx_set_device(0))
    run(**vars(parser.parse_args()))
