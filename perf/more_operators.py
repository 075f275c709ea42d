"""The cases of what stands around the 4-bit cache (include/kmx.h): rotary positions of the rows that go to it, attention over a prompt's own rows, decoding
from a prefix that sequences share, and eviction by accumulated attention weight. What is measured, in its plain form (torch, 32 bits) and through the library.

The cache holds keys and values of `heads` heads in pages of `page` tokens. A block is 16 tokens of one head, 18 dim bytes:
  [0, 8 dim)        codes of the keys: token t, its dim / 2 bytes; channel c = 32 j + 8 g + 4 n + b is nibble n of byte 4 (J g + j) + b
  [8 dim, 16 dim)   codes of the values: pair p, its 16 bytes, one a token; channel c = 32 j + 16 n + i is nibble n of pair 16 j + i
  [16 dim, 17 dim)  scales of the keys, half precision: token t, group j of 32 channels (J = dim / 32 groups)
  [17 dim, 18 dim)  scales of the values: group j, token t
A code is a sign (bit 3) and the index of one of 8 magnitudes that belong to the head and to keys or values; a value is sign * scale * magnitude.
Accumulated weights are floats, [page][head][token of the page].
"""
import importlib
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LEVELS = (0.0381, 0.1172, 0.2036, 0.3003, 0.4097, 0.5396, 0.7075, 0.9712)  # what k-means finds on |x| / max |x| of 32 normal numbers, 8 centroids


# ---------------------------------------------------------------- cases --------------------------

def listed():
    return [
        # the rows of one decoding step of 32 sequences, far into long contexts that the frequencies were stretched for
        dict(name="rotate 32 tokens", op="rotary", tokens=32, query_heads=32, heads=8, dim=128, channels=128, halves=True, inverse=False, stretch=8.0, type="bf16"),
        # a prompt's queries and keys
        dict(name="rotate prompt 16384", op="rotary", tokens=16384, query_heads=32, heads=8, dim=128, channels=128, halves=True, inverse=False, stretch=1.0, type="bf16"),
        # back again (gradients, or rows that get new positions): floats, neighbours in pairs, part of the head
        dict(name="rotate back 5003", op="rotary", tokens=5003, query_heads=10, heads=5, dim=96, channels=64, halves=False, inverse=True, stretch=1.0, type="f32"),
        # a few short prompts that arrived together: latency
        dict(name="prompts 4 x 500", op="prompt", sequences=4, length=500, queries=500, ragged=True, causal=True, query_heads=32, heads=8, dim=128, type="bf16"),
        # one long prompt
        dict(name="prompt 1 x 8192", op="prompt", sequences=1, length=8192, queries=8192, ragged=False, causal=True, query_heads=32, heads=8, dim=128, type="bf16"),
        # prompts of different lengths side by side, three heads to a head of the keys
        dict(name="prompts 6 x 4096", op="prompt", sequences=6, length=4096, queries=4096, ragged=True, causal=True, query_heads=24, heads=8, dim=64, type="f16"),
        # a few answers to the same short instructions: latency
        dict(name="shared 8 x (1000 + 60)", op="shared", groups=1, members=8, prefix=1000, length=60, queries=1, query_heads=32, heads=8, dim=128, page=16, type="bf16"),
        # a full server: 64 sequences behind the same long document
        dict(name="shared 64 x (16384 + 512)", op="shared", groups=1, members=64, prefix=16384, length=512, queries=1, query_heads=64, heads=8, dim=128, page=64, type="bf16"),
        # weights of one decoding step of 32 sequences
        dict(name="weigh 32 x 2048", op="weigh", sequences=32, length=2048, ragged=True, queries=1, query_heads=32, heads=8, dim=128, page=64, type="bf16"),
        # the last queries of a long prompt say what of it is kept
        dict(name="weigh 32 of 32768", op="weigh", sequences=1, length=32768, ragged=False, queries=32, query_heads=32, heads=8, dim=128, page=64, type="bf16"),
        # a cache held at its budget: one token leaves with each that comes
        dict(name="evict 32 x 1025", op="evict", sequences=32, length=1025, ragged=False, heads=8, dim=128, page=64, keep=1024, first=4, recent=32),
        # prompts cut down to their budget
        dict(name="evict 4 x 16384", op="evict", sequences=4, length=16384, ragged=True, heads=8, dim=128, page=64, keep=4096, first=4, recent=64),
    ]


def spread(rng, low, high):
    """A whole number between the two, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "prompt", "prompt", "prompt", "shared", "shared", "weigh", "weigh", "evict", "evict"])
    heads, page = rng.choice([1, 2, 3, 4, 5, 8, 8]), rng.choice([16, 32, 64, 64, 128, 256])
    group, dim = rng.choice([1, 2, 3, 4, 4, 5, 6, 7, 8, 8, 12, 16]), 32 * rng.choice([1, 2, 2, 3, 4, 4, 4, 5, 6, 7, 8])
    kind = rng.choice(["f16", "bf16"])
    if op == "rotary":
        dim = rng.choice([dim, dim, 8 * rng.randint(1, 32)])
        channels = rng.choice([dim, dim, 2 * rng.randint(1, dim // 2)])
        tokens = spread(rng, 1, min(65536, 16384 * 40 * 128 // (heads * (group + 1) * dim)))
        return dict(op=op, tokens=tokens, query_heads=heads * group, heads=heads, dim=dim, channels=channels, halves=rng.random() < 0.5, inverse=rng.random() < 0.3,
                    stretch=rng.choice([1.0, 1.0, 4.0, 8.0, 32.0]), type=rng.choice(["f32", "f16", "bf16"]) if rng.random() < 0.7 else "bf16")
    case = dict(op=op, query_heads=heads * group, heads=heads, dim=dim, type=kind)
    if op == "prompt":
        sequences = spread(rng, 1, 24)
        most = int(math.sqrt(2 ** 36 / (sequences * heads * group * dim)))
        length = spread(rng, 1, max(1, min(8192, most)))
        queries = rng.choice([length, length, length, spread(rng, 1, length)])
        return dict(case, sequences=sequences, length=length, queries=queries, ragged=rng.random() < 0.7, causal=rng.random() < 0.8)
    case["page"] = page
    if op == "shared":
        groups, members, queries = spread(rng, 1, 4), spread(rng, 1, 32), rng.choice([1, 1, 1, 2, 4])
        rows = groups * members * queries * heads * group
        prefix = spread(rng, 1, max(1, min(32768, 2 ** 28 // (groups * heads * dim), 2 ** 29 // rows)))
        return dict(case, groups=groups, members=members, prefix=prefix, length=spread(rng, queries, max(queries, min(2048, 2 ** 28 // (groups * members * heads * dim)))), queries=queries)
    sequences = spread(rng, 1, 32)
    length = spread(rng, 1, max(1, min(65536, 2 ** 27 // (sequences * heads * dim))))
    if op == "weigh":
        queries = min(length, rng.choice([1, 1, 1, 2, 8, 32]), max(1, 2 ** 29 // (sequences * length * heads * group)))
        return dict(case, sequences=sequences, length=length, ragged=rng.random() < 0.7, queries=queries)
    keep = spread(rng, 1, max(1, length))
    first = min(keep, rng.choice([0, 1, 4]))
    del case["query_heads"], case["type"]
    return dict(case, sequences=sequences, length=length, ragged=rng.random() < 0.5, keep=keep, first=first, recent=min(keep - first, rng.choice([0, 1, 8, 64, 300])))


def lengths_of(case):
    """The tokens of each sequence, its queries among them; ragged: from a quarter of the length on, and the sixth of a decoding batch is idle."""
    out, least = [], case.get("queries", 1) if case["op"] != "prompt" else 1
    for b in range(case["sequences"]):
        share = (b * 0.6180339887498949) % 1.0 if case["ragged"] else 0.0
        length = max(least, int(case["length"] * (1.0 - 0.75 * share)), 1)
        out.append(0 if case["ragged"] and b == 5 and least == 1 and case["op"] != "evict" else length)
    return out


def queries_of(case):
    """Queries of each prompt: the last ones of its tokens, where not all are asked for."""
    return [min(n, max(1, int(n * case["queries"] / case["length"]))) for n in lengths_of(case)]


def own_lengths(case):
    """Tokens of each sequence behind a shared prefix: from its queries on to the length."""
    count = case["groups"] * case["members"]
    return [case["queries"] + int((case["length"] - case["queries"]) * ((b * 0.6180339887498949 + 0.5) % 1.0)) for b in range(count)]


def prefix_lengths(case):
    return [max(1, case["prefix"] - case["prefix"] * g // (2 * case["groups"])) for g in range(case["groups"])]


def work(case):
    op, heads, dim = case["op"], case["heads"], case["dim"]
    if op == "evict":
        moved = 0.0
        lengths = lengths_of(case)
        for n in lengths:
            if n > case["keep"]:
                most = n - case["recent"] - case["first"]
                some = case["keep"] - case["recent"] - case["first"]
                moved += case["recent"] + (some * (most - some) / most if most else 0.0)
        return {"bytes": heads * (4 * sum(lengths) + 4 * len(lengths) * case["keep"] + moved * (9 * dim // 4 + 8)), "flops": 0}
    rows_heads = case["query_heads"]
    if op == "rotary":
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": case["tokens"] * (2 * (rows_heads + heads) * dim * size + 4), "flops": 3 * case["tokens"] * (rows_heads + heads) * case["channels"]}
    if op == "prompt":
        n, nq = lengths_of(case), queries_of(case)
        pairs = sum(a * k - a * (a - 1) // 2 if case["causal"] else a * k for a, k in zip(nq, n))
        return {"bytes": sum(nq) * rows_heads * (4 * dim + 4) + 4 * sum(n) * heads * dim, "flops": 4 * pairs * rows_heads * dim}
    held = 9 * dim // 8 * heads  # bytes of a cached token
    nq = case["queries"]
    if op == "shared":
        mine, front = own_lengths(case), prefix_lengths(case)
        pairs = nq * case["members"] * sum(front) + sum(nq * n - nq * (nq - 1) // 2 for n in mine)
        return {"bytes": (sum(mine) + sum(front)) * held + len(mine) * nq * rows_heads * (4 * dim + 4), "flops": 4 * pairs * rows_heads * dim}
    lengths = lengths_of(case)
    pairs = sum(sum(max(0, n - nq + i + 1) for i in range(nq)) for n in lengths)
    return {"bytes": sum(lengths) * (held // 2 + 8 * heads) + len(lengths) * nq * rows_heads * (2 * dim + 4), "flops": 2 * pairs * rows_heads * dim}


# ---------------------------------------------------------------- inputs -------------------------

def rows_of(gen, tokens, heads, dim):
    """Keys and values as a path makes them: keys around a few dozen directions with some channels far larger than the others, values nearly normal."""
    dev = torch.device("cuda")
    centres = torch.randn(48, heads, dim, device=dev, generator=gen)
    which = torch.randint(0, 48, (tokens,), device=dev, generator=gen)
    loud = 1.0 + 3.0 * (torch.rand(heads, dim, device=dev, generator=gen) < 0.04).float()
    keys = (centres[which] + 0.7 * torch.randn(tokens, heads, dim, device=dev, generator=gen)) * loud
    values = torch.randn(tokens, heads, dim, device=dev, generator=gen) * (0.3 + torch.rand(tokens, heads, 1, device=dev, generator=gen))
    return keys, values, centres * loud


def magnitudes(gen, heads):
    """Learned magnitudes of 6 significant bits, a little different for each head and for keys and values."""
    base = torch.tensor(LEVELS, device="cuda").expand(heads, 2, 8)
    part, power = torch.frexp((base * (1.0 + 0.02 * (torch.rand(heads, 2, 8, device="cuda", generator=gen) - 0.5))).clamp(max=1.0))
    return torch.ldexp((part * 64.0).round() / 64.0, power).half().contiguous()


def codes_of(x, levels):
    """x: tokens x heads x dim, levels: heads x 8. The scale of each group of 32 and the code of each value."""
    t, heads, dim = x.shape
    x = x.reshape(t, heads, dim // 32, 32)
    size = x.abs()
    bits = size.amax(-1).view(torch.int32)
    bits = (bits + 0x3FFFF + ((bits >> 19) & 1)) & ~0x7FFFF  # 4 bits behind the point, ties to the even one
    scale = bits.view(torch.float32).clamp(max=63488.0).half()
    middle = (levels[:, :-1].float() + levels[:, 1:].float()) * 0.5
    edges = scale.float()[..., None] * middle[None, :, None, :]
    index = (size[..., None] > edges[..., None, :]).sum(-1, dtype=torch.uint8)
    return scale, (index + 8 * (x < 0).to(torch.uint8)).reshape(t, heads, dim)


def packed(keys, values, levels):
    """The bytes of the codes and the scales, as a block keeps them, for each row."""
    ks, kc = codes_of(keys, levels[:, 0])
    vs, vc = codes_of(values, levels[:, 1])
    t, heads, dim = kc.shape
    kc = kc.reshape(t, heads, dim // 32, 4, 2, 4).permute(0, 1, 3, 2, 4, 5)
    vc = vc.reshape(t, heads, dim // 32, 2, 16)
    kb = (kc[..., 0, :] | (kc[..., 1, :] << 4)).reshape(t, heads, dim // 2)
    vb = (vc[..., 0, :] | (vc[..., 1, :] << 4)).reshape(t, heads, dim // 2)
    return kb, vb, ks, vs


def parts(blocks):
    """Views of blocks (..., 18 dim): codes of keys (..., 16, dim / 2), of values (..., dim / 2, 16), scales of both in half precision (..., 16, dim / 32)."""
    dim = blocks.shape[-1] // 18
    halves = blocks.view(torch.float16)
    return (blocks[..., :8 * dim].unflatten(-1, (16, dim // 2)), blocks[..., 8 * dim:16 * dim].unflatten(-1, (dim // 2, 16)),
            halves[..., 8 * dim:8 * dim + dim // 2].unflatten(-1, (16, dim // 32)), halves[..., 8 * dim + dim // 2:].unflatten(-1, (dim // 32, 16)).transpose(-1, -2))


def fill_cache(s, gen, case, slots, pages):
    """A cache with rows at the given places; what no token has been written to holds anything. The directions of its keys."""
    heads, dim, page = case["heads"], case["dim"], case["page"]
    s["levels"] = magnitudes(gen, heads)
    s["pages"] = pages
    s["blocks"] = torch.full((pages, heads, page // 16, 18 * dim), 255, dtype=torch.uint8, device="cuda")
    step, centres = max(1, 2 ** 26 // (heads * dim)), None
    k, v, sk, sv = parts(s["blocks"])
    for first in range(0, slots.numel(), step):
        at = slots[first:first + step]
        keys, values, centres = rows_of(gen, at.numel(), heads, dim)
        p, b, t = at // page, at % page // 16, at % 16
        k[p, :, b, t], v[p, :, b, :, t], sk[p, :, b, t], sv[p, :, b, t] = packed(keys, values, s["levels"])
    return centres


def queries_for(gen, case, tokens, centres):
    group = case["query_heads"] // case["heads"]
    pick = centres[torch.randint(0, 48, (tokens,), device="cuda", generator=gen)]
    q = 0.35 * pick[:, :, None] + torch.randn(tokens, case["heads"], group, case["dim"], device="cuda", generator=gen)
    return q.reshape(tokens, case["query_heads"], case["dim"]).to(TYPES[case["type"]]).contiguous()


def table_of(gen, lengths, page, pages, where):
    """Pages of some sequences, taken from `where`, and the places of all their tokens in the cache."""
    used = [-(-n // page) for n in lengths]
    width = max(1, max(used))
    there = torch.arange(width, device="cuda")[None, :] < torch.tensor(used, device="cuda")[:, None]
    table = torch.full((len(lengths), width), -1, dtype=torch.int64, device="cuda")
    table[there] = where[:sum(used)]
    at = torch.arange(width * page, device="cuda")
    present = at[None, :] < torch.tensor(lengths, device="cuda")[:, None]
    slots = (table.repeat_interleave(page, 1) * page + at % page)[present]
    return table.int().contiguous(), slots, where[sum(used):]


def pages_for(case, lengths):
    return sum(-(-n // case["page"]) for n in lengths)


def frequencies(case):
    """Radians a position for each pair of channels: those that turn often over the length that was trained on stay, slow ones are stretched. 64 bits."""
    f = 10000.0 ** (-2.0 * torch.arange(case["channels"] // 2, dtype=torch.float64) / case["channels"])
    share = ((8192.0 * f / (2.0 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
    return f * (share + (1.0 - share) / case["stretch"])


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    op, heads, dim = case["op"], case["heads"], case["dim"]
    dev = torch.device("cuda")
    s = {"case": dict(case)}
    if op == "rotary":
        dtype, tokens = TYPES[case["type"]], case["tokens"]
        f = frequencies(case)
        turns = [int(x / (2.0 * math.pi) * 2.0 ** 64) % 2 ** 64 for x in f.tolist()]
        s["frequencies"] = f.to(dev)
        s["turns"] = torch.tensor([x - 2 ** 64 if x >= 2 ** 63 else x for x in turns], dtype=torch.int64, device=dev)  # 64 bits of a turn
        s["gain"] = 1.0 if case["stretch"] == 1.0 else 0.1 * math.log(case["stretch"]) + 1.0
        reach = int(8192 * case["stretch"])
        s["positions"] = (torch.arange(tokens, device=dev) if tokens > 256 else torch.randint(0, reach, (tokens,), device=dev, generator=gen)).int()
        for name, count in (("q", case["query_heads"]), ("k", heads)):
            s[name] = torch.randn(tokens, count, dim, device=dev, generator=gen).to(dtype)
            s[name + "_out"] = torch.empty_like(s[name])
        return s
    if op == "prompt":
        lengths, asked = lengths_of(case), queries_of(case)
        total, rows = sum(lengths), sum(asked)
        keys, values, centres = rows_of(gen, total, heads, dim)
        dtype = TYPES[case["type"]]
        s.update(q=queries_for(gen, case, rows, centres), k=keys.to(dtype), v=values.to(dtype), scale=1.0 / math.sqrt(dim))
        s.update(out=torch.empty_like(s["q"]), lse=torch.empty(rows, case["query_heads"], device=dev), max_queries=max(asked), max_length=max(lengths))
        for name, counts in (("query_starts", asked), ("token_starts", lengths)):
            s[name] = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), device=dev).int()
        return s
    if op == "shared":
        mine, front, nq = own_lengths(case), prefix_lengths(case), case["queries"]
        pages = pages_for(case, mine) + pages_for(case, front) + 2
        where = torch.randperm(pages, device=dev, generator=gen)
        s["prefix_table"], slots, where = table_of(gen, front, case["page"], pages, where)
        s["table"], more, _ = table_of(gen, mine, case["page"], pages, where)
        centres = fill_cache(s, gen, case, torch.cat([slots, more]), pages)
        tokens = len(mine) * nq
        s.update(q=queries_for(gen, case, tokens, centres), scale=1.0 / math.sqrt(dim), max_prefix=max(front), max_length=max(mine))
        s.update(out=torch.empty_like(s["q"]), lse=torch.empty(tokens, case["query_heads"], device=dev), prefix_lengths=torch.tensor(front, device=dev).int(), lengths=torch.tensor(mine, device=dev).int(),
                 prefix_starts=(torch.arange(case["groups"] + 1, device=dev) * nq * case["members"]).int(), starts=(torch.arange(len(mine) + 1, device=dev) * nq).int())
        return s
    lengths = lengths_of(case)
    pages = pages_for(case, lengths) + 2
    s["table"], slots, _ = table_of(gen, lengths, case["page"], pages, torch.randperm(pages, device=dev, generator=gen))
    s.update(lengths=torch.tensor(lengths, device=dev).int(), max_length=max(lengths))
    centres = fill_cache(s, gen, case, slots, pages)
    if op == "weigh":
        nq, tokens = case["queries"], len(lengths) * case["queries"]
        s.update(q=queries_for(gen, case, tokens, centres), scale=1.0 / math.sqrt(dim), starts=(torch.arange(len(lengths) + 1, device=dev) * nq).int())
        s["weights"] = torch.rand(pages, heads, case["page"], device=dev, generator=gen) * 0.05
        score, _ = scores(s, s["table"], s["lengths"], nq, True)
        s["lse"] = torch.logsumexp(score.double(), -1).float().permute(0, 2, 1, 3).reshape(tokens, -1).contiguous()  # what the attention before it left
        return s
    # weights that a while of decoding leaves: most tokens little, a few much; fresh ones none at all (and equal)
    w = torch.exp(2.0 * torch.randn(pages, heads, case["page"], device=dev, generator=gen))
    s["weights"] = torch.where(torch.rand(w.shape, device=dev, generator=gen) < 0.1, torch.zeros_like(w), w)
    s.update(kept=torch.empty(len(lengths), heads, case["keep"], dtype=torch.int32, device=dev), left=torch.empty(len(lengths), dtype=torch.int32, device=dev))
    return s


# ---------------------------------------------------------------- plain form ---------------------

def looked_up(codes, scales, levels):
    """codes, whole rows in the order of the channels (..., heads, dim), scales (..., heads, dim / 32)."""
    heads, dim = codes.shape[-2:]
    table = torch.cat([levels, -levels], -1).float().reshape(-1)
    values = table[codes.int() + 16 * torch.arange(heads, device=codes.device, dtype=torch.int32)[:, None]]
    return (values.unflatten(-1, (dim // 32, 32)) * scales.float()[..., None]).flatten(-2)


def key_rows(kb, ks, levels):
    both = torch.stack([kb & 15, kb >> 4], -1).unflatten(-2, (4, -1, 4))  # g, j, byte, nibble
    return looked_up(both.movedim(-4, -3).movedim(-1, -2).flatten(-4), ks, levels[:, 0])


def value_rows(vb, vs, levels):
    both = torch.stack([vb & 15, vb >> 4], -1).unflatten(-2, (-1, 16))
    return looked_up(both.movedim(-1, -2).flatten(-3), vs, levels[:, 1])


def key_pages(s, table):
    """Keys (sequences, tokens of the table, heads, dim); pages that are not there hold nothing to look at."""
    k, _, sk, _ = parts(s["blocks"][table.clamp(min=0).long()])  # sequences, width, heads, blocks of a page, 16, x
    return key_rows(k.movedim(2, -2).flatten(1, 3), sk.movedim(2, -2).flatten(1, 3), s["levels"])


def value_pages(s, table):
    _, v, _, sv = parts(s["blocks"][table.clamp(min=0).long()])
    return value_rows(v.transpose(-1, -2).movedim(2, -2).flatten(1, 3), sv.movedim(2, -2).flatten(1, 3), s["levels"])


def scores(s, table, lengths, nq, causal):
    """Scores of nq queries each of the table's sequences: sequences, heads, nq, group, tokens, minus infinity where a query does not look, and the tokens that are there."""
    heads, dim = s["case"]["heads"], s["case"]["dim"]
    keys = key_pages(s, table)
    at = torch.arange(keys.shape[1], device=keys.device)
    there = at < lengths[:, None]
    q = s["q"].float().reshape(table.shape[0], nq, heads, -1, dim).permute(0, 2, 1, 3, 4).flatten(2, 3) * s["scale"]
    score = torch.matmul(q, keys.permute(0, 2, 3, 1).contiguous()).unflatten(2, (nq, -1))
    sees = lengths.long()[:, None] - (nq - 1 - torch.arange(nq, device=keys.device)[None, :] if causal else 0)
    return torch.where(at < sees.expand(-1, nq)[:, None, :, None, None], score, -math.inf), there


def plain_rotary(s):
    case = s["case"]
    channels = case["channels"]
    angle = s["positions"].double()[:, None] * s["frequencies"]
    c, sn = (torch.cos(angle) * s["gain"]).float()[:, None], (torch.sin(angle) * s["gain"]).float()[:, None]
    sn = -sn if case["inverse"] else sn

    def turned(x):
        front = x[..., :channels].float()
        a, b = (front[..., :channels // 2], front[..., channels // 2:]) if case["halves"] else (front[..., 0::2], front[..., 1::2])
        both = a * c - b * sn, a * sn + b * c
        front = torch.cat(both, -1) if case["halves"] else torch.stack(both, -1).flatten(-2)
        return torch.cat([front.to(x.dtype), x[..., channels:]], -1)

    return {"q": turned(s["q"]), "k": turned(s["k"])}


def plain_prompt(s):
    case = s["case"]
    heads, dim = case["heads"], case["dim"]
    nq, n = s["query_starts"].diff().long(), s["token_starts"].diff().long()
    i, t = torch.arange(s["max_queries"], device="cuda"), torch.arange(s["max_length"], device="cuda")
    asked, there = i < nq[:, None], t < n[:, None]
    q = s["q"].float()[(s["query_starts"][:-1, None] + i).clamp(max=s["q"].shape[0] - 1)]  # sequences, queries, query heads, dim
    at = (s["token_starts"][:-1, None] + t).clamp(max=s["k"].shape[0] - 1)
    k, v = s["k"].float()[at], torch.where(there[..., None, None], s["v"].float()[at], 0.0)
    q = q.unflatten(2, (heads, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3) * s["scale"]  # sequences, heads, group * queries, dim
    score = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).unflatten(2, (-1, i.numel()))
    sees = n[:, None] - nq[:, None] + i + 1 if case["causal"] else n[:, None].expand(-1, i.numel())
    score = torch.where(t < sees[:, None, None, :, None], score, -math.inf)
    most = score.amax(-1, keepdim=True)
    score = torch.exp(score - torch.where(torch.isfinite(most), most, 0.0))
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.flatten(2, 3), v.permute(0, 2, 1, 3).contiguous()).unflatten(2, (-1, i.numel())) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)[asked]
    return {"out": out.to(s["q"].dtype), "lse": (most + torch.log(total))[..., 0].permute(0, 3, 1, 2).flatten(2, 3)[asked]}


def plain_shared(s):
    case = s["case"]
    heads, dim, nq = case["heads"], case["dim"], case["queries"]
    all_queries = nq * case["members"]
    front, there = scores(s, s["prefix_table"], s["prefix_lengths"], all_queries, False)  # groups, heads, queries of all members, group, tokens
    mine, here = scores(s, s["table"], s["lengths"], nq, True)
    values = torch.where(there[..., None, None], value_pages(s, s["prefix_table"]), 0.0).permute(0, 2, 1, 3).contiguous()
    behind = torch.where(here[..., None, None], value_pages(s, s["table"]), 0.0).permute(0, 2, 1, 3).contiguous()
    apart = lambda x: x.unflatten(2, (case["members"], nq)).movedim(2, 1).flatten(0, 1)  # noqa: E731  to sequences, heads, queries, group, x
    most = torch.maximum(apart(front.amax(-1, keepdim=True)), mine.amax(-1, keepdim=True))
    together = most.unflatten(0, (case["groups"], case["members"])).movedim(1, 2).flatten(2, 3)
    p, r = torch.exp(front - together), torch.exp(mine - most)
    total = apart(p.sum(-1, keepdim=True)) + r.sum(-1, keepdim=True)
    out = apart(torch.matmul(p.flatten(2, 3), values).unflatten(2, (all_queries, -1))) + torch.matmul(r.flatten(2, 3), behind).unflatten(2, (nq, -1))
    out = (out / total).permute(0, 2, 1, 3, 4).reshape(s["q"].shape)
    return {"out": out.to(s["q"].dtype), "lse": (most + torch.log(total))[..., 0].permute(0, 2, 1, 3).reshape(s["q"].shape[:2]).contiguous()}


def plain_weigh(s):
    case = s["case"]
    nq, page = case["queries"], case["page"]
    score, there = scores(s, s["table"], s["lengths"], nq, True)
    lse = s["lse"].reshape(len(score), nq, case["heads"], -1).permute(0, 2, 1, 3)[..., None]
    p = torch.exp(score - lse).sum((2, 3))  # sequences, heads, tokens
    p = torch.where(there[:, None], p, 0.0).unflatten(-1, (-1, page)).transpose(1, 2)  # sequences, pages, heads, tokens of a page
    known = s["table"] >= 0
    s["weights"][s["table"][known].long()] += p[known]
    return {"weights": s["weights"]}


def plain_evict(s):
    case = s["case"]
    heads, page, keep, first, recent = case["heads"], case["page"], case["keep"], case["first"], case["recent"]
    table, n = s["table"].clamp(min=0).long(), s["lengths"].long()[:, None, None]
    weights = s["weights"][table].transpose(1, 2).flatten(2)  # sequences, heads, places of a sequence
    at = torch.arange(weights.shape[2], device="cuda")
    some = keep - first - recent
    rest = (at >= first) & (at < n - recent)
    order = torch.where(rest, weights, -math.inf).sort(dim=-1, descending=True, stable=True)[1]
    rank = torch.empty_like(order).scatter_(2, order, at.expand_as(order))
    cut = n > keep
    stays = torch.where(cut, (at < first) | (rest & (rank < some)) | ((at >= n - recent) & (at < n)), at < n)
    # new places: the recent ones last and in order, of the others those below stay and the rest fills the holes
    edge = torch.where(cut, keep - recent, keep)
    moves = stays & (at >= edge) & (at < n - recent) & cut
    holes = ~stays & (at < edge) & cut
    number = torch.where(holes, holes.cumsum(-1), 0)
    source = torch.full(weights.shape[:2] + (max(keep, at.numel()) + 1,), -1, dtype=torch.int64, device="cuda")
    source[..., 1:at.numel() + 1] = torch.where(stays & (at < edge), at, -1)
    mover = torch.full(weights.shape[:2] + (at.numel() + 1,), -1, dtype=torch.int64, device="cuda")
    mover.scatter_(2, torch.where(moves, moves.cumsum(-1), 0), at.expand_as(order))
    mover[..., 0] = -1
    source[..., 1:at.numel() + 1] = torch.where(holes, mover.gather(2, number), source[..., 1:at.numel() + 1])
    kept = source[..., 1:keep + 1]
    slot = torch.arange(keep, device="cuda")
    kept = torch.where(cut & (slot >= keep - recent), n - keep + slot, kept)
    # rows and their weights
    b, h, to = torch.nonzero((kept >= 0) & (kept != slot), as_tuple=True)
    fr = kept[b, h, to]
    p, u, t = table[b, fr // page], fr % page // 16, fr % 16
    p2, u2, t2 = table[b, to // page], to % page // 16, to % 16
    views = parts(s["blocks"])
    got = [x[p, h, u, t] if i != 1 else x[p, h, u, :, t] for i, x in enumerate(views)]
    for i, (x, y) in enumerate(zip(views, got)):
        if i != 1:
            x[p2, h, u2, t2] = y
        else:
            x[p2, h, u2, :, t2] = y
    s["weights"][p2, h, to % page] = weights[b, h, fr]
    b, h, t = torch.nonzero(cut & (at >= keep) & (at < n) & (s["lengths"][:, None, None] > 0) & torch.ones_like(order, dtype=torch.bool), as_tuple=True)
    s["weights"][table[b, t // page], h, t % page] = 0.0
    return {"kept": kept.int(), "left": s["lengths"].clamp(max=keep), "weights": s["weights"], "blocks": s["blocks"]}


PLAIN = dict(rotary=plain_rotary, prompt=plain_prompt, shared=plain_shared, weigh=plain_weigh, evict=plain_evict)


# ---------------------------------------------------------------- through the library ------------

def handles(s):
    """What a serving program keeps: the cache, the batches and the views of its tensors (addresses and sizes)."""
    km = importlib.import_module("cuda-kmeans_amd")
    case = s["case"]
    see = lambda t: km.DeviceView(t.data_ptr(), t.numel() * t.element_size())  # noqa: E731
    h = {name: see(t) for name, t in s.items() if isinstance(t, torch.Tensor)}
    h["km"] = km
    if "type" in case:
        h["type"] = {"f32": km.TYPE_F32, "f16": km.TYPE_F16, "bf16": km.TYPE_BF16}[case["type"]]
    if case["op"] == "rotary":
        h["rows"] = [km.RotaryRows(h["q"], case["query_heads"], h["q_out"]), km.RotaryRows(h["k"], case["heads"], h["k_out"])]
    elif case["op"] == "prompt":
        h["prompt"] = km.Prompt(case["sequences"], case["query_heads"], case["heads"], case["dim"], s["q"].shape[0], s["k"].shape[0], s["max_queries"], s["max_length"],
                                h["query_starts"], h["token_starts"])
    else:
        h["cache"] = km.Cache4(case["heads"], case["dim"], case["page"], s["pages"], h["levels"], h["blocks"])
        tokens, nq = (s["q"].shape[0], case["queries"]) if "q" in s else (0, 0)
        h["batch"] = km.Cache4Batch(s["table"].shape[0], case.get("query_heads", case["heads"]), tokens, nq, s["max_length"], h.get("starts", h["lengths"]), h["lengths"], h["table"], s["table"].shape[1])
        if case["op"] == "shared":
            h["prefix"] = km.Cache4Batch(case["groups"], case["query_heads"], tokens, nq * case["members"], s["max_prefix"], h["prefix_starts"], h["prefix_lengths"], h["prefix_table"], s["prefix_table"].shape[1])
    return h


def through_library(s):
    case = s["case"]
    h = s.get("handles")
    if h is None:
        h = s["handles"] = handles(s)
    op = case["op"]
    if op == "rotary":
        h["km"].rotary(h["type"], h["rows"], case["tokens"], case["dim"], h["turns"], h["positions"], channels=case["channels"], halves=case["halves"], inverse=case["inverse"], gain=s["gain"])
        return {"q": s["q_out"], "k": s["k_out"]}
    if op == "prompt":
        h["prompt"].attend(h["type"], h["q"], h["k"], h["v"], h["out"], s["scale"], lse=h["lse"], causal=case["causal"])
        return {"out": s["out"], "lse": s["lse"]}
    if op == "shared":
        h["cache"].attend_shared(h["prefix"], h["batch"], h["type"], h["q"], h["out"], s["scale"], lse=h["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if op == "weigh":
        h["cache"].weigh(h["batch"], h["type"], h["q"], h["lse"], h["weights"], s["scale"])
        return {"weights": s["weights"]}
    h["cache"].evict(h["batch"], h["weights"], case["keep"], case["first"], case["recent"], h["kept"], h["left"])
    return {"kept": s["kept"], "left": s["left"], "weights": s["weights"], "blocks": s["blocks"]}  # packed rows move as they are: byte for byte


def run(state):
    return through_library(state) if own else PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------- 64 bits ------------------------

def exact_rows(s, slots, head, which):
    """Rows of one head at the given places, in 64 bits, from where each channel's nibble and scale lie."""
    dim, page = s["case"]["dim"], s["case"]["page"]
    c = torch.arange(dim, device="cuda")
    t = slots % 16
    if which == 0:
        at = t[:, None] * (dim // 2) + ((c % 32 // 8) * (dim // 32) + c // 32) * 4 + c % 4
        shift = 4 * (c // 4 % 2)
    else:
        at = 8 * dim + (16 * (c // 32) + c % 16) * 16 + t[:, None]
        shift = 4 * (c // 16 % 2)
    raw = s["blocks"][slots // page, head, slots % page // 16]
    code = (raw.gather(1, at.expand(len(slots), dim)).long() >> shift) & 15
    place = 16 * dim + 2 * (t[:, None] * (dim // 32) + c // 32) if which == 0 else 17 * dim + 2 * (16 * (c // 32) + t[:, None])
    scale = (raw.gather(1, place).int() + 256 * raw.gather(1, place + 1).int()).to(torch.int16).view(torch.float16).double()
    level = s["levels"][head, which].double()[code % 8]
    return torch.where(code >= 8, -level, level) * scale


def exact_attention(q, k, v, scale, sees):
    """Rows x dim queries of one head, each with the number of tokens it sees: outputs and logarithms of sums."""
    score = q.double() @ k.double().t().contiguous() * scale
    score.masked_fill_(torch.arange(k.shape[0], device="cuda") >= sees[:, None], -math.inf)
    lse = torch.logsumexp(score, -1)
    return torch.exp(score - torch.where(torch.isfinite(lse), lse, 0.0)[:, None]) @ v.double(), lse


def places(table, length, page):
    t = torch.arange(length, device="cuda")
    return table.long()[t // page] * page + t % page


def exact(case, seed):
    s = prepare(case, seed)
    op, heads, dim = case["op"], case["heads"], case["dim"]
    if op == "rotary":
        half = case["channels"] // 2
        angle = s["positions"].double()[:, None] * frequencies(case).cuda()
        turn = torch.polar(torch.full_like(angle, s["gain"]), -angle if case["inverse"] else angle)[:, None]
        out = {}
        for name in ("q", "k"):
            x = s[name].double()
            i = torch.arange(half, device="cuda")
            a, b = (i, i + half) if case["halves"] else (2 * i, 2 * i + 1)
            z = torch.complex(x[..., a], x[..., b]) * turn
            x[..., a], x[..., b] = z.real, z.imag
            out[name] = x
        return out
    if op == "evict":
        # whole numbers and bytes: one sequence and head after the other
        if case["sequences"] * heads > 512 or sum(lengths_of(case)) * heads > 1 << 20:
            return None
        kept, weights = torch.full_like(s["kept"], -1), s["weights"].double()
        for b, n in enumerate(lengths_of(case)):
            at, page = places(s["table"][b], n, case["page"]), case["page"]
            for h in range(heads):
                w = s["weights"][s["table"][b].clamp(min=0).long(), h].reshape(-1)[:n].tolist()
                if n <= case["keep"]:
                    kept[b, h, :n] = torch.arange(n, device="cuda").int()
                    continue
                last = list(range(n - case["recent"], n))
                some = case["keep"] - case["first"] - case["recent"]
                best = sorted(range(case["first"], n - case["recent"]), key=lambda t: (-w[t], t))[:some]
                stay, edge = set(range(case["first"])) | set(best), case["keep"] - case["recent"]
                free = iter(sorted(t for t in stay if t >= edge))
                new = [t if t in stay else next(free) for t in range(edge)] + last
                kept[b, h] = torch.tensor(new, device="cuda").int()
                after = [w[t] for t in new] + [0.0] * (n - case["keep"])
                weights[at // page, h, at % page] = torch.tensor(after, dtype=torch.float64, device="cuda")
        return {"kept": kept, "left": s["lengths"].clamp(max=case["keep"]), "weights": weights, "blocks": None}
    if op == "weigh":
        weights, group = s["weights"].double(), case["query_heads"] // heads
        for b, n in enumerate(lengths_of(case)):
            if n == 0:
                continue
            at = places(s["table"][b], n, case["page"])
            nq = case["queries"]
            sees = (n - nq + 1 + torch.arange(nq, device="cuda")).repeat_interleave(group)
            for h in range(heads):
                rows = slice(b * nq, (b + 1) * nq), slice(h * group, (h + 1) * group)
                score = s["q"][rows].reshape(-1, dim).double() @ exact_rows(s, at, h, 0).t().contiguous() * s["scale"] - s["lse"][rows].reshape(-1, 1).double()
                score.masked_fill_(torch.arange(n, device="cuda") >= sees[:, None], -math.inf)
                weights[at // case["page"], h, at % case["page"]] += torch.exp(score).sum(0)
        return {"weights": weights}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    if op == "prompt":
        group = case["query_heads"] // heads
        first = qfirst = 0
        for n, nq in zip(lengths_of(case), queries_of(case)):
            sees = n - nq + 1 + torch.arange(nq, device="cuda") if case["causal"] else torch.full((nq,), n, device="cuda")
            for h in range(case["query_heads"]):
                k, v = s["k"][first:first + n, h // group], s["v"][first:first + n, h // group]
                out[qfirst:qfirst + nq, h], lse[qfirst:qfirst + nq, h] = exact_attention(s["q"][qfirst:qfirst + nq, h], k, v, s["scale"], sees)
            first, qfirst = first + n, qfirst + nq
        return {"out": out, "lse": lse}
    nq, group = case["queries"], case["query_heads"] // heads
    front, mine = prefix_lengths(case), own_lengths(case)
    if len(mine) * heads > 1024:
        return None
    for h in range(heads):
        for g, length in enumerate(front):
            at = places(s["prefix_table"][g], length, case["page"])
            pk, pv = exact_rows(s, at, h, 0), exact_rows(s, at, h, 1)
            for b in range(g * case["members"], (g + 1) * case["members"]):
                at = places(s["table"][b], mine[b], case["page"])
                k, v = torch.cat([pk, exact_rows(s, at, h, 0)]), torch.cat([pv, exact_rows(s, at, h, 1)])
                rows = slice(b * nq, (b + 1) * nq), slice(h * group, (h + 1) * group)
                sees = (length + mine[b] - nq + 1 + torch.arange(nq, device="cuda")).repeat_interleave(group)
                o, e = exact_attention(s["q"][rows].reshape(-1, dim), k, v, s["scale"], sees)
                out[rows], lse[rows] = o.reshape(nq, group, dim), e.reshape(nq, group)
    return {"out": out, "lse": lse}
