"""Attention operators around a 4-bit paged K/V cache: the cases they are measured on, and their plain forms.

Five operators, in the order a served prompt and its decode steps meet them:

* ``rope``   per-head RMSNorm of queries and keys with the position rotation in the same pass;
* ``prompt`` causal attention of packed sequences of different lengths (grouped heads, window, sinks);
* ``write``  K/V rows quantised to 4 bits into the pages of a cache (read back for the comparison);
* ``read``   a cached range dequantised to packed rows;
* ``cached`` attention of the newest tokens of each sequence over its 4-bit cache.

``run`` computes them in elementary torch operations in 32 bits, or, with ``own`` set, through the
package's public calls.  ``exact`` restates each from its definition in 64 bits.

The cache.  A page holds ``page`` tokens (a power of two from 16) of every K/V head; block_table
[sequences][pages] gives the page of tokens [j * page, (j + 1) * page) of a sequence.  Inside a page each
head has page / 16 blocks of 16 tokens, each 20 * head_dim bytes; with G = head_dim / 32 groups of 32
dims and a code c in 0..15 standing for the value o + d * (16 + c), d and o in f16 per token and group:

* K codes, u32 words [16 tokens][4 t][G w]: dim 32 w + 8 t + 2 n + h is the nibble at bits 4 n + 16 h;
* K scales, f16 [16 tokens][G][d, o];
* V codes, u16 [8 token pairs][head_dim / 16 chunks][4 i][2 tokens]: dim 16 C + 4 i + n of chunk C is
  the nibble at bits 4 n; chunk C of pair p is stored at C ^ ((p & 3) << 1) (C ^ (p & 2) for 64 dims);
* V scales, f16 [8 token pairs][G][d of both tokens, o of both tokens].

Quantising a group: d = f16((max - min) / 15), o = f16(min - 16 d), c = clamp(rint((x - o) / d) - 16, 0, 15),
values clamped to +-16384 first.
"""
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one decode token's heads, straight from the f32 projections (latency)
        dict(name="rope_token", op="rope", tokens=1, heads=32, kv_heads=4, head_dim=128, rot_dim=128,
             interleaved=False, norm=True, src="f32", dst="bf16"),
        # a long prompt of the gated-attention layers: 256-dim heads, 64 of them rotated
        dict(name="rope_prompt", op="rope", tokens=16384, heads=16, kv_heads=2, head_dim=256, rot_dim=64,
             interleaved=False, norm=True, src="bf16", dst="bf16"),
        # short packed prompts of a sliding-window layer with sinks
        dict(name="prompt_packed", op="prompt", seqs=7, longest=301, cached=0, heads=64, kv_heads=8, head_dim=64,
             window=128, sinks=True, src="bf16"),
        # a chunk of new tokens behind a prefix that was read back from the cache
        dict(name="prompt_chunk", op="prompt", seqs=1, longest=2048, cached=9001, heads=16, kv_heads=2,
             head_dim=256, window=0, sinks=False, src="f16"),
        # one whole prompt
        dict(name="prompt_whole", op="prompt", seqs=1, longest=8192, cached=0, heads=32, kv_heads=4, head_dim=128,
             window=0, sinks=False, src="bf16"),
        # one decode step of a batch of 32
        dict(name="write_step", op="write", seqs=32, longest=1, cached=4095, page=16, kv_heads=4, head_dim=128,
             src="bf16"),
        # packed prompts of several sequences, straight from the projections
        dict(name="write_prompt", op="write", seqs=5, longest=8191, cached=0, page=64, kv_heads=8, head_dim=64,
             src="f16"),
        # the cache of one short conversation
        dict(name="read_short", op="read", seqs=1, longest=777, page=32, kv_heads=2, head_dim=256, src="f16"),
        # the prefixes of a batch, before the next chunk's prompt attention
        dict(name="read_prefix", op="read", seqs=8, longest=32768, page=64, kv_heads=4, head_dim=128, src="bf16"),
        # one sequence's decode token at the context that the package's benchmark uses
        dict(name="cached_token", op="cached", seqs=1, longest=4097, fresh=1, page=64, heads=32, kv_heads=4,
             head_dim=128, window=0, sinks=False, src="bf16"),
        # one long context, sinks
        dict(name="cached_long", op="cached", seqs=1, longest=131072, fresh=1, page=64, heads=64, kv_heads=8,
             head_dim=64, window=0, sinks=True, src="f16"),
        # a batch of 32 sequences of different lengths
        dict(name="cached_batch", op="cached", seqs=32, longest=32768, fresh=1, page=16, heads=32, kv_heads=4,
             head_dim=128, window=0, sinks=False, src="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["rope", "prompt", "write", "read", "cached", "cached", "prompt"])
    kv_heads, rep, hd = rng.choice([(8, 8, 64), (4, 8, 128), (2, 8, 256), (4, 4, 128), (2, 2, 64), (5, 1, 128),
                                    (1, 16, 128), (3, 3, 64), (2, 5, 256)])
    src = rng.choice(["bf16", "f16"])
    page = rng.choice([16, 32, 64, 128])
    if op == "rope":
        return dict(op=op, tokens=_spread(rng, 1, 16384), heads=kv_heads * rep, kv_heads=kv_heads, head_dim=hd,
                    rot_dim=rng.choice([hd, hd // 2, hd // 4]), interleaved=rng.random() < 0.4,
                    norm=rng.random() < 0.7, src=rng.choice(["f32", "bf16", "f16"]), dst=src)
    if op == "prompt":
        seqs = _spread(rng, 1, 12)
        longest = _spread(rng, 1, 4096 if seqs == 1 else 1024)
        cached = rng.choice([0, 0, _spread(rng, 1, 4000)])
        return dict(op=op, seqs=seqs, longest=longest, cached=cached, heads=kv_heads * rep, kv_heads=kv_heads,
                    head_dim=hd, window=rng.choice([0, 0, 128, _spread(rng, 1, 2000)]), sinks=rng.random() < 0.4,
                    src=src)
    if op == "write":
        seqs = _spread(rng, 1, 32)
        return dict(op=op, seqs=seqs, longest=_spread(rng, 1, 16384 // seqs), cached=rng.choice([0, _spread(rng, 1, 5000)]),
                    page=page, kv_heads=kv_heads, head_dim=hd, src=rng.choice(["bf16", "f16", "f32"]))
    if op == "read":
        seqs = _spread(rng, 1, 16)
        return dict(op=op, seqs=seqs, longest=_spread(rng, 1, 131072 // seqs), page=page, kv_heads=kv_heads,
                    head_dim=hd, src=src)
    seqs = _spread(rng, 1, 32)
    fresh = rng.choice([1, 1, 1, 2, 4])
    return dict(op=op, seqs=seqs, longest=_spread(rng, fresh, 262144 // seqs), fresh=fresh, page=page,
                heads=kv_heads * rep, kv_heads=kv_heads, head_dim=hd,
                window=rng.choice([0, 0, 0, 128, _spread(rng, 1, 4000)]), sinks=rng.random() < 0.4, src=src)


def _lens(case, longest, shortest=1):
    """The sequences' lengths: the first is the longest, the others spread over the logarithm."""
    r = random.Random(case["seqs"] * 1000003 + longest)
    return [longest] + [_spread(r, shortest, longest) for _ in range(case["seqs"] - 1)]


def _shapes(case):
    """(new tokens, tokens already cached) of every sequence."""
    if case["op"] == "read":
        n = _lens(case, case["longest"])
        return n, [0] * len(n)
    if case["op"] == "cached":
        n = _lens(case, case["longest"], max(case["fresh"], case["longest"] // 64))
        return [case["fresh"]] * len(n), [x - case["fresh"] for x in n]
    new = _lens(case, case["longest"])
    return new, (_lens(case, case["cached"]) if case["cached"] else [0] * len(new))


def _pairs(new, old, window):
    """How many (query, key) pairs causal attention of new tokens behind old ones has."""
    total = 0
    for n, c in zip(new, old):
        if window <= 0 or window >= c + n:
            total += n * c + n * (n + 1) // 2
        else:
            full = max(0, min(n, window - c))                     # queries that see every earlier key
            total += full * c + full * (full + 1) // 2 + (n - full) * window
    return total


def work(case):
    hd, kv = case["head_dim"], case["kv_heads"]
    if case["op"] == "rope":
        rows = case["tokens"] * (case["heads"] + kv)
        return {"bytes": rows * hd * (BYTES[case["src"]] + BYTES[case["dst"]]) + case["tokens"] * (4 * case["rot_dim"] + 4)
                + 8 * hd, "flops": rows * (4 * hd + 3 * case["rot_dim"])}
    new, old = _shapes(case)
    n, token4 = sum(new), kv * hd * 5 // 4                        # K and V of one token: 4 bits + f16 d, o per 32
    size = BYTES[case["src"]]
    if case["op"] == "write":                                     # rows in, blocks out, and read back once
        return {"bytes": n * (2 * kv * hd * (size + 2) + 2 * token4), "flops": n * kv * hd * 10}
    if case["op"] == "read":
        return {"bytes": n * (token4 + 2 * kv * hd * size), "flops": n * kv * hd * 4}
    H, window = case["heads"], case["window"]
    flops = 4 * hd * H * _pairs(new, old, window)
    if case["op"] == "prompt":
        return {"bytes": size * hd * (2 * n * H + 2 * kv * (n + sum(old))), "flops": flops}
    seen = [min(a + b, window + a - 1) if window > 0 else a + b for a, b in zip(new, old)]
    return {"bytes": sum(seen) * token4 + 2 * size * hd * H * n, "flops": flops}


# ---------------------------------------------------------------- inputs

def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cum(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def _values(gen, n, heads, hd):
    """K or V rows as the projections make them: unit spread, with an offset for each channel."""
    x = torch.randn(n, heads, hd, device="cuda", generator=gen)
    return x.add_(0.3 * torch.randn(heads, hd, device="cuda", generator=gen))


def _new_cache(case, gen, lens):
    """Pages in a shuffled pool (some unused, all with what an earlier user left) and the block table."""
    page, hd, kv = case["page"], case["head_dim"], case["kv_heads"]
    per = [-(-x // page) for x in lens]
    pool = sum(per) + 3
    order = torch.randperm(pool, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(per)), -1, dtype=torch.int32, device="cuda")
    for i, (a, n) in enumerate(zip(_cum(per), per)):
        table[i, :n] = order[a:a + n]
    pages = torch.randint(0, 256, (pool, kv, page // 16, 20 * hd), dtype=torch.uint8, device="cuda", generator=gen)
    return pages, table


def _fill(case, s, gen, cum, start):
    """What earlier steps cached: random rows, quantised into the pages."""
    n = cum[-1]
    step = max(1, (1 << 27) // (case["kv_heads"] * case["head_dim"]))
    c, b = _i32(cum), _i32(start)
    for a in range(0, n, step):
        m = min(step, n - a)
        at = torch.arange(a, a + m, device="cuda")
        place = _places(case, s["table"], c, b, at)
        rows = [_values(gen, m, case["kv_heads"], case["head_dim"]) for _ in range(2)]
        _plain_write(case, s["pages"], place, *rows)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    hd, kv = case["head_dim"], case["kv_heads"]
    s = {"case": case}
    if case["op"] == "rope":
        T, H, rot = case["tokens"], case["heads"], case["rot_dim"]
        t = TYPES[case["src"]]
        s["qkv"] = torch.randn(T, (H + 2 * kv) * hd, device="cuda", generator=gen).to(t)
        s["q"] = s["qkv"][:, :H * hd].unflatten(1, (H, hd))
        s["k"] = s["qkv"][:, H * hd:(H + kv) * hd].unflatten(1, (kv, hd))
        s["q_norm"], s["k_norm"] = ((1 + 0.1 * torch.randn(hd, device="cuda", generator=gen)) if case["norm"] else None
                                    for _ in range(2))
        most = T + 4096
        ang = torch.arange(most, device="cuda", dtype=torch.float64)[:, None] * torch.pow(
            1e6, -torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        first = int(torch.randint(0, 4096, (1,), device="cuda", generator=gen))
        s["pos"] = torch.arange(first, first + T, device="cuda", dtype=torch.int32)
        s["q_out"] = torch.empty(T, H, hd, device="cuda", dtype=TYPES[case["dst"]])
        s["k_out"] = torch.empty(T, kv, hd, device="cuda", dtype=TYPES[case["dst"]])
        return s
    t = TYPES[case["src"]]
    new, old = _shapes(case)
    n, both = sum(new), [a + b for a, b in zip(new, old)]
    if case["op"] == "prompt":
        H = case["heads"]
        s["q"] = (1.7 * torch.randn(n, H, hd, device="cuda", generator=gen)).to(t)
        s["k"] = _values(gen, sum(both), kv, hd).to(t)
        wide = _values(gen, sum(both), 2 * kv, hd).to(t)          # v is the second half of a wider row
        s["v"] = wide[:, kv:]
        s["cu_q"], s["cu_k"] = _i32(_cum(new)), _i32(_cum(both))
        s["sinks"] = torch.randn(H, device="cuda", generator=gen) if case["sinks"] else None
        s["out"] = torch.empty(n, H, hd, device="cuda", dtype=t)
        s["max_q"], s["max_k"] = max(new), max(both)
        return s
    s["pages"], s["table"] = _new_cache(case, gen, both)
    if case["op"] == "write":
        s["k"] = _values(gen, n, kv, hd).to(t)
        wide = _values(gen, n, 2 * kv, hd).to(t)
        s["v"] = wide[:, kv:]
        s["cu"], s["start"] = _i32(_cum(new)), _i32(old)
        back = torch.bfloat16 if case["src"] == "bf16" else torch.float16
    else:
        _fill(case, s, gen, _cum(both), [0] * len(both))
        s["cu"], s["start"] = _i32(_cum(both)), _i32([0] * len(both))
        n, back = sum(both), t
    if case["op"] == "cached":
        B, F, H = case["seqs"], case["fresh"], case["heads"]
        s["q"] = (1.7 * torch.randn(B, F, H, hd, device="cuda", generator=gen)).to(t)
        s["lens"], s["longest"] = _i32(both), max(both)
        s["sinks"] = torch.randn(H, device="cuda", generator=gen) if case["sinks"] else None
        s["out"] = torch.empty_like(s["q"])
    else:
        s["k_back"], s["v_back"] = (torch.empty(n, kv, hd, device="cuda", dtype=back) for _ in range(2))
    return s


# ---------------------------------------------------------------- plain forms

def _places(case, table, cu, start, at):
    """Where packed rows `at` of the sequences cu stand in the pages: index arrays into the pages seen as
    words (K codes) and as 16-bit halves (everything else)."""
    seq = torch.searchsorted(cu, at.to(torch.int32), right=True) - 1
    return _places_of(case, table, seq, at - cu[seq] + start[seq])


def _places_of(case, table, seq, pos):
    hd, kv, page = case["head_dim"], case["kv_heads"], case["page"]
    G = hd // 32
    dev = pos.device
    pos = pos.long()
    num = table[seq, pos // page].long()
    base = ((num[:, None] * kv + torch.arange(kv, device=dev)) * (page // 16) + (pos % page // 16)[:, None]) * (20 * hd)
    tok = (pos % 16)[:, None]
    pair, par = tok // 2, tok % 2
    g = torch.arange(G, device=dev)
    k_word = (base // 4 + tok * 4 * G)[..., None] + torch.arange(4 * G, device=dev)
    k_scale = (base // 2 + 4 * hd + tok * 2 * G)[..., None] + 2 * g
    twist = (pair & 2) if hd == 64 else (pair & 3) << 1
    chunk = torch.arange(hd // 16, device=dev) ^ twist[..., None]
    v_half = (base // 2 + 5 * hd + par)[..., None] + (pair[..., None] * (hd // 16) + chunk) * 8
    v_half = v_half[..., None] + 2 * torch.arange(4, device=dev)
    v_scale = (base // 2 + 9 * hd + par + pair * 4 * G)[..., None] + 4 * g
    return k_word, k_scale, v_half, v_scale


def _codes(x):
    """Rows [n][heads][hd] -> codes and the f16 d and o of their groups of 32 dims."""
    x = torch.where(torch.isnan(x), torch.zeros_like(x), x).clamp(-16384.0, 16384.0).unflatten(2, (-1, 32))
    lo, hi = x.amin(-1), x.amax(-1)
    d = ((hi - lo) / 15.0).half()
    o = (lo - 16.0 * d.float()).half()
    df = d.float()[..., None]
    c = torch.round((x - o.float()[..., None]) / df) - 16.0
    c = torch.where(df > 0, c, torch.zeros_like(c)).clamp(0.0, 15.0).to(torch.int32)
    return c, d, o


def _plain_write(case, pages, place, k, v):
    k_word, k_scale, v_half, v_scale = place
    words, halves = pages.view(torch.int32).view(-1), pages.view(torch.int16).view(-1)
    low = torch.arange(4, device=pages.device, dtype=torch.int32) * 4
    c, d, o = _codes(k.float())                                   # [n][heads][G][32 = 4 t, 4 n, 2 h]
    shift = low[:, None] + torch.arange(2, device=pages.device, dtype=torch.int32) * 16
    w = (c.unflatten(3, (4, 4, 2)) << shift).sum((4, 5), dtype=torch.int32)
    words[k_word] = w.transpose(2, 3).flatten(2)
    halves[k_scale], halves[k_scale + 1] = d.view(torch.int16), o.view(torch.int16)
    c, d, o = _codes(v.float())
    h = (c.flatten(2).unflatten(2, (-1, 4, 4)) << low).sum(4, dtype=torch.int32)
    halves[v_half] = h.to(torch.int16)
    halves[v_scale], halves[v_scale + 2] = d.view(torch.int16), o.view(torch.int16)


def _plain_read(case, pages, place):
    """(k, v) rows [n][heads][hd] in 32 bits."""
    k_word, k_scale, v_half, v_scale = place
    words, halves = pages.view(torch.int32).view(-1), pages.view(torch.int16).view(-1)
    low = torch.arange(4, device=pages.device, dtype=torch.int32) * 4
    shift = low[:, None] + torch.arange(2, device=pages.device, dtype=torch.int32) * 16
    w = words[k_word].unflatten(2, (4, -1)).transpose(2, 3)       # [n][heads][w][t]
    k = ((w[..., None, None] >> shift) & 15).flatten(3).float()
    f16 = lambda i: halves[i].view(torch.float16).float()[..., None]
    k = (k + 16.0) * f16(k_scale) + f16(k_scale + 1)
    h = halves[v_half].to(torch.int32)
    v = ((h[..., None] >> low) & 15).flatten(2).unflatten(2, (-1, 32)).float()
    v = (v + 16.0) * f16(v_scale) + f16(v_scale + 2)
    return k.flatten(2), v.flatten(2)


def _plain_rope(s):
    case, out = s["case"], []
    rot = case["rot_dim"]
    cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]

    def one(x, w):
        x = x.float()
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        r, rest = x[..., :rot], x[..., rot:]
        if case["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = r[..., :rot // 2], r[..., rot // 2:]
            r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((r, rest), -1).to(TYPES[case["dst"]])

    return one(s["q"], s["q_norm"]), one(s["k"], s["k_norm"])


def _plain_attention(q, k, v, q_pos, keys, window, sinks):
    """q [b][nq][H][hd], k / v [b][nk][kv][hd] in 32 bits; q_pos [b][nq] each query's place among its keys,
    keys [b] how many of them there are.  A query without keys gives zeros."""
    b, nq, H, hd = q.shape
    kv = k.shape[2]
    q = q.unflatten(2, (kv, H // kv)).permute(0, 2, 3, 1, 4).flatten(2, 3)        # [b][kv][rep * nq][hd]
    sc = (q @ k.permute(0, 2, 3, 1)).mul_(hd ** -0.5)
    sc = sc.unflatten(2, (H // kv, nq))
    j = torch.arange(k.shape[1], device=q.device)
    ok = (j <= q_pos[..., None]) & (j < keys[:, None, None])
    if window > 0:
        ok = ok & (j > q_pos[..., None] - window)
    sc.masked_fill_(~ok[:, None, None], float("-inf"))
    m = sc.amax(-1, keepdim=True)
    if sinks is not None:
        m = torch.maximum(m, sinks.view(kv, -1)[None, :, :, None, None])
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = sc.sub_(m).exp_()
    den = p.sum(-1, keepdim=True)
    if sinks is not None:
        den = den + torch.exp(sinks.view(kv, -1)[None, :, :, None, None] - m)
    o = (p.flatten(2, 3) @ v.permute(0, 2, 1, 3)).unflatten(2, (H // kv, nq))
    o = o / torch.where(den > 0, den, torch.ones_like(den))
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3)                                 # [b][nq][H][hd]


def _padded(cu, most):
    """Packed rows as [sequences][most]: each place's row, and whether it is one."""
    at = torch.arange(most, device=cu.device)
    n = cu[1:] - cu[:-1]
    ok = at < n[:, None]
    return torch.where(ok, cu[:-1, None] + at, 0), ok, n


def _plain_prompt(s):
    case = s["case"]
    qi, q_ok, nq = _padded(s["cu_q"], s["max_q"])
    ki, k_ok, nk = _padded(s["cu_k"], s["max_k"])
    k, v = s["k"].float()[ki], s["v"].float()[ki]
    v = torch.where(k_ok[..., None, None], v, 0.0)
    place = (nk - nq)[:, None] + torch.arange(s["max_q"], device=ki.device)
    o = _plain_attention(s["q"].float()[qi], k, v, place, nk, case["window"], s["sinks"])
    return o[q_ok].to(s["q"].dtype)


def _plain_cached(s):
    case = s["case"]
    B, F = case["seqs"], case["fresh"]
    at = torch.arange(s["longest"], device="cuda")
    at = torch.minimum(at, s["lens"][:, None] - 1)
    seq = torch.arange(B, device="cuda")[:, None].expand_as(at).flatten()
    k, v = _plain_read(case, s["pages"], _places_of(case, s["table"], seq, at.flatten()))
    place = s["lens"][:, None] - F + torch.arange(F, device="cuda")
    o = _plain_attention(s["q"].float(), k.unflatten(0, (B, -1)), v.unflatten(0, (B, -1)), place, s["lens"],
                         case["window"], s["sinks"])
    return o.to(s["q"].dtype)


# ---------------------------------------------------------------- the package's calls

_contexts = {}


def _context():
    """The program's context, on torch's current stream."""
    if "one" not in _contexts:
        from moe_stream_b200 import Context
        _contexts["one"] = Context(0, stream=torch.cuda.current_stream())
    return _contexts["one"]


def _cache(s):
    """The handle that a program keeps for its cache."""
    if "cache" not in s:
        from moe_stream_b200 import KV4Cache
        s["cache"] = KV4Cache(s["pages"], s["table"], s["case"]["kv_heads"], s["case"]["head_dim"], s["case"]["page"])
    return s["cache"]


def run(s):
    case = s["case"]
    op = case["op"]
    if op == "rope":
        if not own:
            return _plain_rope(s)
        _context().qk_norm_rope(s["q"], s["k"], s["q_norm"], s["k_norm"], 1e-6, s["cos"], s["sin"], s["pos"],
                                s["q_out"], s["k_out"], interleaved=case["interleaved"])
        return s["q_out"], s["k_out"]
    if op == "prompt":
        if not own:
            return _plain_prompt(s)
        _context().prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], s["out"], window=case["window"],
                                    sinks=s["sinks"])
        return s["out"]
    if op == "cached":
        if not own:
            return _plain_cached(s)
        if "work" not in s:                                       # a program keeps its workspace
            n = _context().kv4_attention_workspace_bytes(_cache(s), case["seqs"], case["fresh"], case["heads"])
            s["work"] = torch.empty(n, dtype=torch.uint8, device="cuda")
        _context().kv4_attention(_cache(s), s["q"], s["lens"], s["out"], s["work"], window=case["window"],
                                 sinks=s["sinks"])
        return s["out"]
    if not own:
        place = _places(case, s["table"], s["cu"], s["start"], torch.arange(s["k_back"].shape[0], device="cuda"))
        if op == "write":
            _plain_write(case, s["pages"], place, s["k"], s["v"])
        k, v = _plain_read(case, s["pages"], place)
        return k.to(s["k_back"].dtype), v.to(s["v_back"].dtype)
    if op == "write":
        _context().kv4_write(_cache(s), s["k"], s["v"], s["cu"], s["start"])
    _context().kv4_read(_cache(s), s["cu"], s["start"], s["k_back"], s["v_back"])
    return s["k_back"], s["v_back"]


# ---------------------------------------------------------------- from the definitions, in 64 bits

def _exact_values(case, pages, table, seq, n):
    """K and V of the first n tokens of a sequence in 64 bits, nibble by nibble from their byte addresses."""
    hd, kv, page = case["head_dim"], case["kv_heads"], case["page"]
    G, raw = hd // 32, pages.reshape(-1)
    p = torch.arange(n, device=raw.device)
    block = (table[seq].long()[p // page] * kv * (page // 16))[:, None, None] + (torch.arange(kv, device=raw.device)
                                                                                 * (page // 16))[:, None]
    block = (block + (p % page // 16)[:, None, None]) * (20 * hd)  # [n][kv][1]
    tok = (p % 16)[:, None, None]
    dim = torch.arange(hd, device=raw.device)
    w, t, m, h = dim // 32, dim % 32 // 8, dim % 8 // 2, dim % 2

    def nibble(byte, odd):
        return (raw[byte].to(torch.int64) >> (4 * odd)) & 15

    def f16(byte):
        both = raw[byte].to(torch.int64) | (raw[byte + 1].to(torch.int64) << 8)
        return both.to(torch.int16).view(torch.float16).double()

    code = nibble(block + tok * (hd // 2) + (t * G + w) * 4 + m // 2 + 2 * h, m % 2)
    at = block + 8 * hd + (tok * G + w) * 4
    k = f16(at + 2) + f16(at) * (16 + code)
    chunk = dim // 16
    twist = (tok // 2 % 4 // 2) * 2 if hd == 64 else (tok // 2 % 4) * 2
    u16 = ((tok // 2) * (hd // 16) + torch.bitwise_xor(chunk, twist)) * 8 + dim % 16 // 4 * 2 + tok % 2
    code = nibble(block + 10 * hd + u16 * 2 + dim % 4 // 2, dim % 2)
    at = block + 18 * hd + ((tok // 2) * G + w) * 8 + 2 * (tok % 2)
    return k, f16(at + 4) + f16(at) * (16 + code)


def _exact_quantised(x):
    """What 4 bits keep of rows [n][heads][hd]."""
    x = x.double().nan_to_num(0.0, 1e30, -1e30).clamp(-16384, 16384)
    out = torch.empty_like(x)
    for a in range(0, x.shape[2], 32):
        g = x[..., a:a + 32]
        low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        d = ((high - low) / 15).half().double()
        o = (low - 16 * d).half().double()
        c = torch.where(d > 0, ((g - o) / torch.where(d > 0, d, 1.0)).round() - 16, 0.0).clamp(0, 15)
        out[..., a:a + 32] = o + d * (16 + c)
    return out


def _exact_rows(q, k, v, place, window, sink):
    """softmax(q k^T / sqrt(hd)) v of one head; place [nq]: the index of each query's own key."""
    sc = q @ k.T / q.shape[1] ** 0.5
    j = torch.arange(k.shape[0], device=q.device)
    hidden = j > place[:, None]
    if window > 0:
        hidden |= j <= place[:, None] - window
    sc[hidden] = float("-inf")
    full = sc if sink is None else torch.cat((sc, sink.expand(sc.shape[0], 1)), 1)
    log = torch.logsumexp(full, 1, keepdim=True)
    return torch.exp(sc - torch.where(torch.isinf(log), 0.0, log)) @ v


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        got = []
        rot = case["rot_dim"]
        turn = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]
        for x, w in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])):
            x = x.double()
            if w is not None:
                x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w.double()
            y = x.clone()
            ia = torch.arange(0, rot, 2, device="cuda") if case["interleaved"] else torch.arange(rot // 2, device="cuda")
            ib = ia + 1 if case["interleaved"] else ia + rot // 2
            z = torch.complex(x[..., ia], x[..., ib]) * turn
            y[..., ia], y[..., ib] = z.real, z.imag
            got.append(y)
        return tuple(got)
    new, old = _shapes(case)
    if op == "write":
        return _exact_quantised(s["k"]), _exact_quantised(s["v"])
    if op == "read":
        got = [_exact_values(case, s["pages"], s["table"], i, n) for i, n in enumerate(new)]
        return torch.cat([a for a, _ in got]), torch.cat([b for _, b in got])
    rep = case["heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    at_q = at_k = 0
    for i, (n, c) in enumerate(zip(new, old)):
        if op == "prompt":
            q, o = s["q"][at_q:at_q + n], out[at_q:at_q + n]
            k, v = s["k"][at_k:at_k + n + c].double(), s["v"][at_k:at_k + n + c].double()
            at_q, at_k = at_q + n, at_k + n + c
        else:
            q, o = s["q"][i], out[i]
            k, v = _exact_values(case, s["pages"], s["table"], i, n + c)
        place = c + torch.arange(n, device="cuda")
        for h in range(case["heads"]):
            o[:, h] = _exact_rows(q[:, h].double(), k[:, h // rep], v[:, h // rep], place, case["window"],
                                  None if s["sinks"] is None else s["sinks"][h].double())
    return out
