"""GPU tests of the attention operators of ragged batches against plain restatements in 64 bits.

Tolerances (u = half a step of the output type: 2^-8 bf16, 2^-11 f16, 2^-24 f32):
* rotation: the f32 chain has at most 24 roundings on |a| + |b| of a value's pair (16 squares and 5 partial sums
  of the mean halved by the root, then the quotient, two products and the rotation's products and sum), then u;
* cache: d, o and codes are IEEE f32 operations, so the pages are compared byte for byte; reading back is one f32
  rounding and u;
* attention: with A = sum p |v| / sum p, the probabilities' rounding costs up to w A (w = u of the element type, or
  of f16 over the 4-bit cache, whose dequantised v adds another 2^-11 A), an error e of the scores up to 2 e A (the
  numerator and the denominator), and the f32 sums, exp2 and rescalings 2^-14 A; then u |out|.
"""
import numpy as np
import pytest

from . import attn_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}   # one subnormal step


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from moe_stream_b200.engine import Context
    c = Context(0)
    c.set_stream(torch.cuda.current_stream())
    yield c
    c.close()


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cum(v):
    return [0] + list(np.cumsum(v))


def within(got, want, tol):
    got, want = got.double(), want.double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float((got - want).abs()[bad].max()), float((got - want).abs().div(tol)[bad].max()),
                           bad.nonzero()[0].tolist())


# ---------------------------------------------------------------- norms and rotation

ROPE = [  # tokens, heads, kv_heads, hd, rot, interleaved, norm, src, dst
    (1, 32, 4, 128, 128, False, True, "float32", "bfloat16"),
    (7, 64, 8, 64, 64, False, False, "bfloat16", "bfloat16"),
    (33, 16, 2, 256, 64, False, True, "float16", "float16"),
    (5, 3, 1, 64, 32, True, True, "float32", "float32"),
    (130, 5, 5, 128, 48, True, True, "bfloat16", "float16"),
    (3, 2, 1, 96, 96, False, True, "float32", "float32"),       # no vector path
    (4, 3, 2, 34, 10, True, True, "float16", "float32"),
    (2, 1, 1, 512, 512, False, True, "bfloat16", "bfloat16"),
    (6, 4, 2, 128, 6, False, False, "float32", "bfloat16"),
    (4100, 32, 4, 128, 128, False, True, "bfloat16", "bfloat16"),
    (4100, 16, 3, 64, 64, True, True, "float32", "float16"),
    (2050, 16, 2, 256, 64, False, True, "float32", "bfloat16"),
]


def rope_inputs(T, H, kv, hd, rot, norm, src, seed=0, pad=0):
    g = gen(seed)
    qkv = torch.randn(T, (H + 2 * kv) * hd + pad, device="cuda", generator=g).to(src)
    q, k = qkv[:, :H * hd].unflatten(1, (H, hd)), qkv[:, H * hd:(H + kv) * hd].unflatten(1, (kv, hd))
    w = [1 + 0.2 * torch.randn(hd, device="cuda", generator=g) for _ in range(2)] if norm else [None, None]
    ang = torch.arange(T + 40, device="cuda", dtype=torch.float64)[:, None] * torch.pow(
        1e4, -torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    pos = torch.randint(0, T + 40, (T,), device="cuda", generator=g).to(torch.int32)
    return qkv, q, k, w[0], w[1], ang.cos().float(), ang.sin().float(), pos


@pytest.mark.parametrize("case", ROPE, ids=str)
def test_qk_norm_rope(ctx, case):
    T, H, kv, hd, rot, inter, norm, src, dst = case
    src, dst = getattr(torch, src), getattr(torch, dst)
    _, q, k, qw, kw, cos, sin, pos = rope_inputs(T, H, kv, hd, rot, norm, src, seed=T, pad=8 if T == 7 else 0)
    qo, ko = torch.empty(T, H, hd, dtype=dst, device="cuda"), torch.empty(T, kv, hd, dtype=dst, device="cuda")
    ctx.qk_norm_rope(q, k, qw, kw, 1e-6, cos, sin, pos, qo, ko, interleaved=inter)
    ctx.sync()
    for x, w, got in ((q, qw, qo), (k, kw, ko)):
        want, size = R.rope(x, w, 1e-6, cos, sin, pos, inter)
        within(got, want, HALF[dst] * want.abs() + 24 * 2.0 ** -24 * size * (1 + HALF[dst]) + TINY[dst])


def test_qk_norm_rope_in_place_strided_and_zero_rows(ctx):
    qkv, q, k, qw, kw, cos, sin, pos = rope_inputs(19, 8, 2, 128, 64, True, torch.bfloat16, seed=3)
    q[4], k[5] = 0, 0                                            # eps keeps a row of zeros at zero
    want = [R.rope(x, w, 1e-5, cos, sin, pos, False) for x, w in ((q, qw), (k, kw))]
    v = qkv[:, 10 * 128:].clone()
    ctx.qk_norm_rope(q, k, qw, kw, 1e-5, cos, sin, pos, q, k)
    ctx.sync()
    for got, (y, size) in zip((q, k), want):
        within(got, y, HALF[torch.bfloat16] * y.abs() + 25 * 2.0 ** -24 * size + TINY[torch.bfloat16])
    assert torch.equal(qkv[:, 10 * 128:], v)


@pytest.mark.parametrize("hd", [128, 96])
def test_qk_norm_rope_bad_position_is_skipped_and_reported(ctx, hd):
    from moe_stream_b200._lib import MsError
    _, q, k, qw, kw, cos, sin, pos = rope_inputs(6, 4, 2, hd, 32, True, torch.float32, seed=5)
    pos[2], pos[4] = -1, cos.shape[0]
    qo, ko = torch.full_like(q.contiguous(), 7.0), torch.full_like(k.contiguous(), 7.0)
    ctx.qk_norm_rope(q, k, qw, kw, 1e-6, cos, sin, pos, qo, ko)
    with pytest.raises(MsError) as e:
        ctx.sync()
    assert e.value.status == 11
    ctx.sync()
    for got in (qo, ko):
        assert (got[[2, 4]] == 7.0).all() and (got[[0, 1, 3, 5]] != 7.0).any()


def test_no_rows_is_no_work(ctx):
    from moe_stream_b200.engine import KV4Cache
    e = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="cuda")
    t = torch.ones(4, 32, device="cuda")
    ctx.qk_norm_rope(e(0, 4, 64), e(0, 2, 64), None, None, 1e-6, t, t, i32([]), e(0, 4, 64), e(0, 2, 64))
    ctx.prompt_attention(e(0, 4, 64), e(0, 2, 64), e(0, 2, 64), i32([0]), i32([0]), e(0, 4, 64))
    ctx.prompt_attention(e(0, 4, 64), e(0, 2, 64), e(0, 2, 64), i32([0, 0]), i32([0, 0]), e(0, 4, 64))
    cache = KV4Cache(torch.zeros(KV4Cache.page_bytes(2, 64, 16), dtype=torch.uint8, device="cuda"), i32([[0]]), 2, 64, 16)
    ctx.kv4_write(cache, e(0, 2, 64), e(0, 2, 64), i32([0, 0]), i32([0]))
    ctx.kv4_read(cache, i32([0, 0]), i32([0]), e(0, 2, 64), e(0, 2, 64))
    ctx.sync()


# ---------------------------------------------------------------- the 4-bit cache

def new_cache(lens, page, kv, hd, seed, fill=None):
    """A shuffled pool with three pages that nobody has, and its handle."""
    from moe_stream_b200.engine import KV4Cache
    r = np.random.default_rng(seed)
    per = [-(-n // page) for n in lens]
    pool = sum(per) + 3
    order = r.permutation(pool)
    table = np.full((len(lens), max(per + [1])), -1, np.int32)
    for i, (a, n) in enumerate(zip(cum(per), per)):
        table[i, :n] = order[a:a + n]
    raw = r.integers(0, 256, (pool, kv, page // 16, R.block_bytes(hd)), dtype=np.uint8)
    if fill is not None:
        raw[:] = fill
    pages = torch.from_numpy(raw).cuda()
    return KV4Cache(pages, torch.from_numpy(table).cuda(), kv, hd, page), raw.copy(), table


CACHE = [  # new, start, page, kv, hd, type
    ([1], [0], 16, 1, 64, "bfloat16"),
    ([1, 1, 1], [15, 16, 4], 16, 2, 128, "float16"),
    ([5, 0, 20, 1], [3, 9, 13, 0], 16, 2, 64, "float32"),
    ([33, 2], [1, 30], 32, 1, 128, "bfloat16"),
    ([17, 18], [0, 63], 64, 3, 256, "float16"),
    ([2, 3, 4, 5, 6, 7], [1, 1, 2, 2, 3, 3], 128, 1, 64, "bfloat16"),
    ([1] * 32, [5 * i % 33 for i in range(32)], 16, 1, 64, "float16"),
    ([7 * i * i % 5 for i in range(77)], [3 * i % 19 for i in range(77)], 16, 1, 64, "float16"),
    ([0] * 40 + [3] + [0] * 20 + [1], [2] * 62, 16, 2, 64, "bfloat16"),
    ([2 + i % 2 for i in range(300)], [i % 3 for i in range(300)], 16, 1, 64, "bfloat16"),
]


@pytest.mark.parametrize("case", CACHE, ids=str)
def test_kv4_write_and_read(ctx, case):
    new, start, page, kv, hd, t = case
    t = getattr(torch, t)
    cache, raw, table = new_cache([a + b for a, b in zip(new, start)], page, kv, hd, seed=hd + len(new))
    n, g = sum(new), gen(hd + page)
    k = (torch.randn(n, kv, hd, device="cuda", generator=g) * 3).to(t)
    v = torch.randn(n + 2, 2 * kv, hd, device="cuda", generator=g).to(t)[:, kv:]   # rows behind the last, strided
    k = torch.cat((k, torch.full((2, kv, hd), 5.0, dtype=t, device="cuda")))
    k[0, 0, :32] = 1.5                                            # a constant group: d = 0
    cu, st = i32(cum(new)), i32(start)
    ctx.kv4_write(cache, k, v, cu, st)
    ctx.sync()
    kn, vn = k.float().cpu().numpy(), v.float().cpu().numpy()
    for i, (a, m) in enumerate(zip(cum(new), new)):
        for j in range(m):
            R.put_token(raw, table, i, start[i] + j, page, kv, hd, kn[a + j], vn[a + j])
    assert np.array_equal(cache.pages.cpu().numpy(), raw)        # every other byte as it was
    out = [torch.full((n + 2, kv, hd), 9.0, dtype=ty, device="cuda") for ty in (t, t)]
    ctx.kv4_read(cache, cu, st, *out)
    ctx.sync()
    for i, (a, m) in enumerate(zip(cum(new), new)):
        if not m:
            continue
        vals = R.cache_values(raw, table, i, start[i] + m, page, kv, hd)
        for got, want, x, d, o in ((out[0], vals[0], kn, vals[2], vals[3]), (out[1], vals[1], vn, vals[4], vals[5])):
            want, d, o = (torch.from_numpy(np.ascontiguousarray(z[start[i]:])).cuda() for z in (want, d, o))
            within(got[a:a + m], want, (HALF[t] + 2.0 ** -24) * want.abs() + TINY[t])
            # half a step, and where d or o were rounded to f16 the ends of the range move by that
            x = torch.from_numpy(x[a:a + m]).cuda().double()
            within(want, x, d * (0.5 + 2.0 ** -18) + 31 * d * 2.0 ** -11 + o.abs() * 2.0 ** -11 + 2.0 ** -20)
    assert (out[0][n:] == 9.0).all() and (out[1][n:] == 9.0).all()


@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("t", ["float32", "bfloat16", "float16"])
def test_kv4_write_values_half_way_between_codes(ctx, t, hd):
    """Groups from 0 to 30 steps with 15 intervals: every odd value is a tie, which goes to the even code."""
    t = getattr(torch, t)
    cache, raw, table = new_cache([48], 16, 2, hd, seed=3)
    r = np.random.default_rng(4)
    x = r.integers(0, 31, (48, 2, hd // 32, 32)).astype(np.float32)
    x[..., 0], x[..., 1] = 0, 30
    x = r.permuted(x, axis=-1) - r.integers(0, 31, (48, 2, hd // 32, 1))
    x *= 2.0 ** r.integers(-9, 9, (48, 2, hd // 32, 1)).astype(np.float32)
    if t == torch.float32:                                            # and values next to the ties
        x = np.where(r.random(x.shape) < 0.5, x, np.nextafter(x, np.float32(1e9) * r.choice([-1, 1], x.shape), dtype=np.float32))
    k = torch.from_numpy(x.reshape(48, 2, hd).astype(np.float32)).cuda().to(t)
    v = k.flip(0).contiguous()
    ctx.kv4_write(cache, k, v, i32([0, 48]), i32([0]))
    ctx.sync()
    for j in range(48):
        R.put_token(raw, table, 0, j, 16, 2, hd, k[j].float().cpu().numpy(), v[j].float().cpu().numpy())
    assert np.array_equal(cache.pages.cpu().numpy(), raw)


@pytest.mark.parametrize("t", ["float32", "bfloat16", "float16"])
def test_kv4_write_unusual_values(ctx, t):
    t = getattr(torch, t)
    cache, raw, table = new_cache([16], 16, 1, 64, seed=1, fill=0xFF)
    k = torch.randn(16, 1, 64, device="cuda", generator=gen(2))
    k[0, 0, 3], k[1, 0, 7], k[2, 0, 9] = float("nan"), float("inf"), float("-inf")
    k[3] *= 1e-7
    k[4] *= 1e-4
    k[5] = 100 + 0.01 * k[5]
    k[6, 0, :32], k[6, 0, 32:] = float("nan"), 0
    k[7] *= 6000
    if t != torch.float16:
        k[8] *= 1e20
    k = k.to(t)
    v = k.flip(0).contiguous()
    ctx.kv4_write(cache, k, v, i32([0, 16]), i32([0]))
    ctx.sync()
    for j in range(16):
        R.put_token(raw, table, 0, j, 16, 1, 64, k[j].float().cpu().numpy(), v[j].float().cpu().numpy())
    assert np.array_equal(cache.pages.cpu().numpy(), raw)
    back = [torch.empty_like(k) for _ in range(2)]
    ctx.kv4_read(cache, i32([0, 16]), i32([0]), *back)
    ctx.sync()
    assert all(torch.isfinite(b).all() for b in back)


def test_kv4_bad_pages_and_positions_are_skipped_and_reported(ctx):
    from moe_stream_b200._lib import MsError
    cache, raw, table = new_cache([48, 48], 16, 2, 64, seed=4)
    cache.block_table[0, 1], cache.block_table[1, 0] = cache.args.n_pages, -7
    k = torch.randn(96, 2, 64, device="cuda", generator=gen(1)).half()
    cu, st = i32([0, 48, 96]), i32([0, 8])                       # sequence 1 also runs past its table
    ctx.kv4_write(cache, k, k, cu, st)
    with pytest.raises(MsError) as e:
        ctx.sync()
    assert e.value.status == 11
    kn = k.float().cpu().numpy()
    for i, a, s in ((0, 0, 0), (1, 48, 8)):
        for j in range(48):
            p = s + j
            if p // 16 < 3 and (i, p // 16) not in ((0, 1), (1, 0)):
                R.put_token(raw, table, i, p, 16, 2, 64, kn[a + j], kn[a + j])
    assert np.array_equal(cache.pages.cpu().numpy(), raw)
    out = [torch.full_like(k, 9.0) for _ in range(2)]
    ctx.kv4_read(cache, cu, st, *out)
    with pytest.raises(MsError):
        ctx.sync()
    skipped = [j for j in range(16, 32)] + [48 + j for j in range(48) if 8 + j < 16 or 8 + j >= 48]
    kept = [j for j in range(96) if j not in skipped]
    for o in out:
        assert (o[skipped] == 9.0).all() and (o[kept] != 9.0).any(-1).all()


# ---------------------------------------------------------------- attention over the cache

def fill_cache(ctx, cache, lens, seed, scale=1.0, t=torch.bfloat16):
    n = sum(lens)
    g = gen(seed)
    kv, hd = cache.kv_heads, cache.head_dim
    k = torch.randn(n, kv, hd, device="cuda", generator=g) + 0.3 * torch.randn(kv, hd, device="cuda", generator=g)
    v = torch.randn(n, kv, hd, device="cuda", generator=g) + 0.3 * torch.randn(kv, hd, device="cuda", generator=g)
    ctx.kv4_write(cache, k.to(t), (v * scale).to(t), i32(cum(lens)), i32([0] * len(lens)))
    ctx.sync()


def cached_reference(cache, table, q, lens, window, scale, sinks):
    """(want, tolerance) of every row."""
    raw = cache.pages.cpu().numpy()
    B, F, H, hd = q.shape
    want, tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    rep, u = H // cache.kv_heads, HALF[q.dtype]
    for i, n in enumerate(lens):
        if not n:
            continue
        k, v, dk, ok, dv, ov = (torch.from_numpy(x).cuda() for x in R.cache_values(raw, table, i, n, cache.page_tokens, cache.kv_heads, hd))
        place = n - F + torch.arange(F, device="cuda")
        o, A = R.attention(q[i], k, v, place, window, scale, sinks)
        # scores: 32 products q (16 + c) of a group in f32 steps, the group's d and o applied in f32
        qa = q[i].double().abs()
        e = torch.einsum("fhd,mhd->hfm", qa, (32 * 31 * 2 * dk + 8 * ok.abs()).repeat_interleave(rep, 1)) * scale * 2.0 ** -24
        e = e.amax(-1).T[..., None] + 2.0 ** -23 * torch.einsum("fhd,mhd->hfm", qa, k.abs().repeat_interleave(rep, 1)).amax(-1).T[..., None] * scale
        want[i], tol[i] = o, u * o.abs() + (1 + u) * (2 * 2.0 ** -11 + 2 * e + 2.0 ** -14) * A + TINY[q.dtype] + 2.0 ** -22 * dv.amax()
    return want, tol


CACHED = [  # lens, n_query, page, heads, kv, hd, window, sinks, type
    ([1], 1, 16, 8, 1, 64, 0, False, "bfloat16"),
    ([1, 2, 17, 31, 32, 33], 1, 16, 16, 2, 128, 0, False, "bfloat16"),
    ([0, 5, 100, 0, 64], 1, 16, 64, 8, 64, 0, True, "float16"),
    ([700, 3, 129], 1, 64, 16, 2, 256, 0, False, "float16"),
    ([700, 3, 129, 128, 127], 1, 32, 32, 4, 128, 128, True, "bfloat16"),
    ([1000, 40, 4], 4, 64, 8, 1, 64, 0, False, "bfloat16"),
    ([300, 7], 3, 128, 15, 3, 128, 20, True, "float16"),
    ([77, 513], 1, 16, 4, 4, 256, 0, False, "bfloat16"),
    ([77, 513], 5, 32, 6, 2, 64, 1, False, "bfloat16"),
    ([260], 8, 16, 32, 2, 128, 0, False, "float16"),
    ([5000], 1, 64, 8, 1, 128, 0, False, "bfloat16"),
    ([9000, 20], 2, 64, 16, 2, 64, 4000, True, "float16"),
    ([3, 2, 9], 9, 16, 8, 2, 64, 0, True, "bfloat16"),           # lengths below n_query: leading queries have no tokens
    ([64] * 200, 1, 16, 8, 2, 64, 0, False, "bfloat16"),
]


def cached_case(ctx, case, poison, seed=0):
    lens, F, page, H, kv, hd, window, sinks, t = case
    t = getattr(torch, t)
    cache, _, table = new_cache(lens, page, kv, hd, seed=len(lens) + hd, fill=0xFF if poison else 0x3C)
    fill_cache(ctx, cache, lens, seed + 1)
    g = gen(seed + 2)
    q = (1.5 * torch.randn(len(lens), F, H, hd, device="cuda", generator=g)).to(t)
    sk = torch.randn(H, device="cuda", generator=g) if sinks else None
    out = torch.full_like(q, 7.0)
    work = torch.empty(ctx.kv4_attention_workspace_bytes(cache, len(lens), F, H), dtype=torch.uint8, device="cuda").fill_(255)
    return cache, table, q, i32(lens), out, work, window, sk


@pytest.mark.parametrize("case", CACHED, ids=str)
def test_kv4_attention(ctx, case):
    """The unused tokens of every page and the pages of nobody hold NaN scales."""
    cache, table, q, lens, out, work, window, sk = cached_case(ctx, case, poison=True)
    ctx.kv4_attention(cache, q, lens, out, work, window=window, sinks=sk)
    ctx.sync()
    want, tol = cached_reference(cache, table, q, case[0], window, case[5] ** -0.5, sk)
    within(out, want, tol)
    again = torch.empty_like(out)
    ctx.kv4_attention(cache, q, lens, again, work, window=window, sinks=sk)
    ctx.sync()
    assert torch.equal(out, again)


def test_kv4_attention_sharp_and_flat_scores_own_scale(ctx):
    case = ([400, 1500], 1, 64, 16, 2, 128, 0, True, "bfloat16")
    cache, table, q, lens, out, work, window, sk = cached_case(ctx, case, poison=True)
    for scale, shift in ((1.0, 0.0), (1e-4, 0.0), (0.2, 30.0), (0.2, -60.0)):
        s = sk + shift
        ctx.kv4_attention(cache, q, lens, out, work, sinks=s, scale=scale)
        ctx.sync()
        want, tol = cached_reference(cache, table, q, case[0], 0, scale, s)
        within(out, want, tol)


def test_kv4_attention_bad_pages_and_lengths(ctx):
    from moe_stream_b200._lib import MsError
    case = ([100, 90, 80], 1, 16, 8, 1, 64, 0, False, "float16")
    cache, table, q, lens, out, work, _, _ = cached_case(ctx, case, poison=False)
    cache.block_table[0, 3] = cache.args.n_pages + 5
    lens[1] = -4
    lens[2] = 16 * cache.args.max_pages + 1
    cache.block_table[2, 5:] = -1
    ctx.kv4_attention(cache, q, lens, out, work)
    with pytest.raises(MsError) as e:
        ctx.sync()
    assert e.value.status == 11
    assert (out[1] == 0).all() and torch.isfinite(out[0]).all() and torch.isfinite(out[2]).all()


# ---------------------------------------------------------------- prompt attention

PROMPT = [  # new, cached, heads, kv, hd, window, sinks, type
    ([1], [0], 8, 1, 64, 0, False, "bfloat16"),
    ([1, 2, 3, 0, 127, 128, 129], [0] * 7, 16, 2, 128, 0, False, "bfloat16"),
    ([5, 300, 1], [0, 0, 0], 64, 8, 64, 128, True, "bfloat16"),
    ([257], [0], 16, 2, 256, 0, False, "float16"),
    ([33, 70], [500, 3], 16, 2, 256, 0, True, "bfloat16"),
    ([100, 1, 64], [129, 1000, 0], 12, 4, 128, 50, False, "float16"),
    ([40, 41], [7, 0], 5, 5, 64, 1, False, "float16"),
    ([130], [0], 10, 2, 256, 17, True, "float16"),
    ([65], [200], 128, 1, 64, 0, False, "bfloat16"),
    ([65, 66], [200, 0], 100, 1, 128, 60, True, "bfloat16"),
    ([700], [0], 8, 8, 128, 0, False, "bfloat16"),
    ([3] * 150, [2] * 150, 8, 2, 64, 0, False, "bfloat16"),
    ([1500], [333], 8, 1, 64, 0, True, "float16"),
    ([600, 600], [0, 900], 14, 2, 128, 256, False, "bfloat16"),
]


def prompt_reference(q, k, v, new, both, window, scale, sinks):
    want, tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    rep, u = q.shape[1] // k.shape[1], HALF[q.dtype]
    a = b = 0
    for n, m in zip(new, both):
        if n:
            place = m - n + torch.arange(n, device="cuda")
            kk, vv = k[b:b + m], v[b:b + m]
            o, A = R.attention(q[a:a + n], kk, vv, place, window, scale, sinks)
            e = torch.einsum("fhd,mhd->hfm", q[a:a + n].double().abs(), kk.double().abs().repeat_interleave(rep, 1))
            e = (e.amax(-1) if m else e.sum(-1)).T[..., None] * scale * 2.0 ** -23 * q.shape[2] ** 0.5 * 4
            want[a:a + n], tol[a:a + n] = o, u * o.abs() + (1 + u) * (u + 2 * e + 2.0 ** -14) * A + TINY[q.dtype]
        a, b = a + n, b + m
    return want, tol


def prompt_case(new, cached, H, kv, hd, t, seed=0, behind=3):
    """Packed rows, v strided, with `behind` rows of NaN in front of nothing: they follow the last sequence."""
    g = gen(seed)
    both = [a + b for a, b in zip(new, cached)]
    q = (1.5 * torch.randn(sum(new) + behind, H, hd, device="cuda", generator=g)).to(t)
    k = torch.randn(sum(both) + behind, kv, hd, device="cuda", generator=g).to(t)
    v = (torch.randn(sum(both) + behind, 2 * kv, hd, device="cuda", generator=g) + 0.2).to(t)[:, kv:]
    for x, n in ((q, sum(new)), (k, sum(both)), (v, sum(both))):
        x[n:] = float("nan")
    return q, k, v, i32(cum(new)), i32(cum(both)), both, g


@pytest.mark.parametrize("case", PROMPT, ids=str)
def test_prompt_attention(ctx, case):
    new, cached, H, kv, hd, window, sinks, t = case
    q, k, v, cq, ck, both, g = prompt_case(new, cached, H, kv, hd, getattr(torch, t), seed=hd + H)
    sk = torch.randn(H, device="cuda", generator=g) if sinks else None
    out = torch.full((q.shape[0], H + 1, hd), 7.0, dtype=q.dtype, device="cuda")[:, :H]
    ctx.prompt_attention(q, k, v, cq, ck, out, window=window, sinks=sk)
    ctx.sync()
    n = sum(new)
    want, tol = prompt_reference(q[:n], k, v, new, both, window, hd ** -0.5, sk)
    within(out[:n], want, tol)
    assert (out[n:] == 7.0).all()
    again = torch.empty_like(out)
    ctx.prompt_attention(q, k, v, cq, ck, again, window=window, sinks=sk)
    ctx.sync()
    assert torch.equal(out[:n], again[:n])


@pytest.mark.parametrize("hd,H,kv,n,cached", [(64, 16, 2, 700, 900), (128, 8, 8, 900, 1300), (256, 16, 2, 700, 900)])
def test_prompt_attention_gives_the_same_bits_every_time(ctx, hd, H, kv, n, cached):
    """Many key tiles, sharp scores (the running maximum rises often): every product and rescaling is waited for."""
    q, k, v, cq, ck, both, _ = prompt_case([n], [cached], H, kv, hd, torch.bfloat16, seed=6, behind=0)
    q = q * 2
    first = torch.empty_like(q)
    ctx.prompt_attention(q, k, v, cq, ck, first)
    ctx.sync()
    want, tol = prompt_reference(q, k, v, [n], both, 0, hd ** -0.5, None)
    within(first, want, tol)
    for _ in range(40):
        out = torch.empty_like(q)
        ctx.prompt_attention(q, k, v, cq, ck, out)
        assert torch.equal(out, first)


def test_prompt_attention_neighbours_hold_nan_and_infinity(ctx):
    """What another sequence holds does not reach a sequence's rows."""
    new, H, kv, hd = [70, 90, 50], 8, 2, 128
    for bad in (0, 1, 2):
        q, k, v, cq, ck, both, _ = prompt_case(new, [0, 0, 0], H, kv, hd, torch.bfloat16, seed=9)
        c = cum(new)
        want, tol = prompt_reference(q[:210], k, v, new, both, 0, hd ** -0.5, None)
        for x, val in ((q, float("nan")), (k, float("nan")), (v, float("inf"))):
            x[c[bad]:c[bad + 1]] = val
        out = torch.empty_like(q)
        ctx.prompt_attention(q, k, v, cq, ck, out)
        ctx.sync()
        keep = [j for i in range(3) if i != bad for j in range(c[i], c[i + 1])]
        within(out[keep], want[keep], tol[keep])


def test_prompt_attention_more_queries_than_keys(ctx):
    """The first queries of a sequence that has fewer keys than queries see none: zeros, with sinks too."""
    q, k, v, _, _, _, g = prompt_case([40, 30], [0, 0], 8, 2, 64, torch.float16, seed=4)
    cq, ck = i32([0, 40, 70]), i32([0, 25, 25])
    sk = torch.randn(8, device="cuda", generator=g)
    for s in (None, sk):
        out = torch.full_like(q, 7.0)
        ctx.prompt_attention(q, k, v, cq, ck, out, sinks=s)
        ctx.sync()
        want, tol = prompt_reference(q[:70], k[:25], v[:25], [40, 30], [25, 0], 0, 0.125, s)
        within(out[:70], want, tol)
        assert (out[:15] == 0).all() and (out[40:70] == 0).all()


def test_prompt_attention_bad_offsets_are_reported(ctx):
    from moe_stream_b200._lib import MsError
    q, k, v, _, _, _, _ = prompt_case([20, 20], [0, 0], 8, 2, 64, torch.float16, seed=4)
    out = torch.full_like(q, 7.0)
    ctx.prompt_attention(q, k, v, i32([0, 20, 40]), i32([0, 20, 4000]), out)
    with pytest.raises(MsError) as e:
        ctx.sync()
    assert e.value.status == 11
    assert (out[20:] == 7.0).all() and (out[:20] != 7.0).any()


# ---------------------------------------------------------------- far offsets, wide windows, infinite sinks, two streams

def far_rows(rows, heads, hd, t, stride=1 << 22):
    """[rows, heads, hd] whose last rows lie beyond 2^32 bytes: a view with a wide stride."""
    base = torch.empty((rows - 1) * stride + heads * hd, dtype=t, device="cuda")
    return base.as_strided((rows, heads, hd), (stride, hd, 1))


def test_offsets_beyond_32_bits(ctx):
    """1030 rows 2^22 elements apart span 8.6 GB; the cache's pool has 5 GB of pages, the last ones in use."""
    from moe_stream_b200.engine import KV4Cache
    n, H, kv, hd, t = 1030, 4, 2, 64, torch.bfloat16
    g = gen(1)
    near = lambda heads: torch.randn(n, heads, hd, device="cuda", generator=g).to(t)
    q, k, v = near(H), near(kv), near(kv)
    cos, sin = torch.ones(n, 32, device="cuda"), torch.zeros(n, 32, device="cuda")
    far = far_rows(n, H, hd, t)
    far.copy_(q)
    ko = torch.empty_like(k)
    ctx.qk_norm_rope(far, k, None, None, 0.0, cos, sin, torch.arange(n, device="cuda", dtype=torch.int32), far, ko)
    ctx.sync()
    assert torch.equal(far, q) and torch.equal(ko, k)
    cu, out = i32([0, n]), torch.empty_like(q)
    ctx.prompt_attention(q, k, v, cu, cu, out)
    ctx.prompt_attention(far, k, v, cu, cu, far_out := far_rows(n, H, hd, t))
    ctx.sync()
    assert torch.equal(out, far_out)
    del far_out
    fk = far_rows(n, kv, hd, t)
    fk.copy_(k)
    again = torch.empty_like(out)
    ctx.prompt_attention(q, fk, v, cu, cu, again)
    ctx.sync()
    assert torch.equal(out, again)
    per = KV4Cache.page_bytes(kv, hd, 16)
    pool = (5 << 30) // per
    pages = torch.empty(pool * per, dtype=torch.uint8, device="cuda")
    need = -(-n // 16)
    table = torch.arange(pool - need, pool, dtype=torch.int32, device="cuda")[None]
    cache = KV4Cache(pages, table, kv, hd, 16)
    ctx.kv4_write(cache, fk, v, cu, i32([0]))
    small = KV4Cache(pages[(pool - need) * per:].clone(), torch.arange(need, dtype=torch.int32, device="cuda")[None], kv, hd, 16)
    o = [torch.empty(1, 1, H, hd, dtype=t, device="cuda") for _ in range(2)]
    for c, x in zip((cache, small), o):
        work = torch.empty(ctx.kv4_attention_workspace_bytes(c, 1, 1, H), dtype=torch.uint8, device="cuda")
        ctx.kv4_attention(c, q[:1, None].contiguous(), i32([n]), x, work)
        ctx.sync()
    assert torch.equal(*o)
    back = [torch.empty(n, kv, hd, dtype=t, device="cuda") for _ in range(2)]
    ctx.kv4_read(cache, cu, i32([0]), fk, back[1])
    ctx.kv4_read(small, cu, i32([0]), back[0], back[1])
    ctx.sync()
    assert torch.equal(fk, back[0])


def test_windows_wider_than_anything(ctx):
    """The largest window is no window."""
    case = ([100, 30], 2, 16, 8, 1, 64, 0, False, "bfloat16")
    cache, table, q, lens, out, work, _, _ = cached_case(ctx, case, poison=True)
    ctx.kv4_attention(cache, q, lens, out, work)
    wide = torch.empty_like(out)
    ctx.kv4_attention(cache, q, lens, wide, work, window=2 ** 31 - 1)
    pq, pk, pv, cq, ck, _, _ = prompt_case([70, 40], [0, 9], 8, 2, 64, torch.bfloat16)
    po = [torch.empty_like(pq) for _ in range(2)]
    ctx.prompt_attention(pq, pk, pv, cq, ck, po[0])
    ctx.prompt_attention(pq, pk, pv, cq, ck, po[1], window=2 ** 31 - 1)
    ctx.sync()
    assert torch.equal(out, wide) and torch.equal(po[0][:110], po[1][:110])


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_infinite_sinks(ctx, hd):
    """A sink of -infinity is none, one of +infinity takes everything."""
    H = 8
    case = ([300, 0, 41], 1, 16, H, 2, hd, 0, False, "float16")
    cache, table, q, lens, out, work, _, _ = cached_case(ctx, case, poison=True)
    pq, pk, pv, cq, ck, _, _ = prompt_case([70, 40], [0, 9], H, 2, hd, torch.float16)
    sk = torch.full((H,), float("-inf"), device="cuda")
    sk[3] = float("inf")
    so, ps, po = torch.empty_like(out), torch.empty_like(pq), torch.empty_like(pq)
    ctx.kv4_attention(cache, q, lens, out, work)
    ctx.kv4_attention(cache, q, lens, so, work, sinks=sk)
    ctx.prompt_attention(pq, pk, pv, cq, ck, po)
    ctx.prompt_attention(pq, pk, pv, cq, ck, ps, sinks=sk)
    ctx.sync()
    keep = [h for h in range(H) if h != 3]
    assert (so[:, :, 3] == 0).all() and torch.equal(so[:, :, keep], out[:, :, keep])
    assert (ps[:110, 3] == 0).all() and torch.equal(ps[:110, keep], po[:110, keep])


def test_two_streams_at_once(ctx):
    """Both attentions running on two streams, each call with its own workspace and outputs."""
    from moe_stream_b200.engine import Context
    streams = [torch.cuda.Stream() for _ in range(2)]
    cs = [Context(0, stream=s) for s in streams]
    sets = []
    for i, hd in enumerate((64, 128, 256)):
        case = ([3000, 200, 17], 1, 32, 16, 2, hd, 0, False, "bfloat16")
        kv = cached_case(ctx, case, poison=True, seed=i)
        pr = prompt_case([300, 90], [100, 0], 16, 2, hd, torch.bfloat16, seed=i)
        want = torch.empty_like(kv[4]), torch.empty_like(pr[0])
        ctx.kv4_attention(kv[0], kv[2], kv[3], want[0], kv[5])
        ctx.prompt_attention(*pr[:5], want[1])
        sets.append((kv, pr, want))
    ctx.sync()
    torch.cuda.synchronize()
    outs = []
    for r in range(10):
        for c in cs:
            for kv, pr, want in sets:
                o = torch.full_like(kv[4], 7.0), torch.full_like(pr[0], 7.0), torch.empty_like(kv[5])
                outs.append((o, want))
    torch.cuda.synchronize()
    k = 0
    for r in range(10):
        for c in cs:
            for kv, pr, want in sets:
                o = outs[k][0]
                k += 1
                c.kv4_attention(kv[0], kv[2], kv[3], o[0], o[2])
                c.prompt_attention(*pr[:5], o[1])
    for c in cs:
        c.sync()
    for o, want in outs:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1][:390], want[1][:390])
    for c in cs:
        c.close()


# ---------------------------------------------------------------- together

def test_chain_prompt_then_decode(ctx):
    """Projections -> norm and rotation -> prompt attention, and the rows into the cache; then decode steps over the
    cache, and a second chunk of the prompt behind the prefix that was read back."""
    H, kv, hd, page, t = 16, 2, 128, 16, torch.bfloat16
    lens, steps = [37, 90], 3
    total = [n + steps for n in lens]
    cache, raw, table = new_cache(total, page, kv, hd, seed=8, fill=0xFF)
    qkv, q, k, qw, kw, cos, sin, _ = rope_inputs(sum(lens), H, kv, hd, hd, True, torch.float32, seed=2)
    v = qkv[:, (H + kv) * hd:].unflatten(1, (kv, hd))
    pos = i32([j for n in lens for j in range(n)])
    qr, kr = torch.empty(sum(lens), H, hd, dtype=t, device="cuda"), torch.empty(sum(lens), kv, hd, dtype=t, device="cuda")
    cu, zero = i32(cum(lens)), i32([0, 0])
    out = torch.empty_like(qr)
    vb = v.to(t)
    ctx.qk_norm_rope(q, k, qw, kw, 1e-6, cos, sin, pos, qr, kr)
    ctx.prompt_attention(qr, kr, vb, cu, cu, out)
    ctx.kv4_write(cache, kr, vb, cu, zero)
    ctx.sync()
    want, tol = prompt_reference(qr, kr, vb, lens, lens, 0, hd ** -0.5, None)
    within(out, want, tol)
    # the second half of each prompt as a chunk behind its cached prefix
    half = [n // 2 for n in lens]
    prefix = [torch.empty(sum(half), kv, hd, dtype=t, device="cuda") for _ in range(2)]
    ctx.kv4_read(cache, i32(cum(half)), zero, *prefix)
    rows = [torch.cat([torch.cat((p[a:a + h], x[b + h:b + n])) for a, b, h, n in zip(cum(half), cum(lens), half, lens)])
            for p, x in zip(prefix, (kr, vb))]
    tail = [n - h for n, h in zip(lens, half)]
    qt = torch.cat([qr[b + h:b + n] for b, h, n in zip(cum(lens), half, lens)])
    ot = torch.empty_like(qt)
    ctx.prompt_attention(qt, rows[0], rows[1], i32(cum(tail)), cu, ot)
    ctx.sync()
    want, tol = prompt_reference(qt, rows[0], rows[1], tail, lens, 0, hd ** -0.5, None)
    within(ot, want, tol)
    # decode: one token per sequence and step
    work = torch.empty(ctx.kv4_attention_workspace_bytes(cache, 2, 1, H), dtype=torch.uint8, device="cuda")
    for s in range(steps):
        qkv, q, k, _, _, _, _, _ = rope_inputs(2, H, kv, hd, hd, True, torch.float32, seed=20 + s)
        v = qkv[:, (H + kv) * hd:].unflatten(1, (kv, hd))
        at = [n + s for n in lens]
        qr, kr = torch.empty(2, H, hd, dtype=t, device="cuda"), torch.empty(2, kv, hd, dtype=t, device="cuda")
        ctx.qk_norm_rope(q, k, qw, kw, 1e-6, cos, sin, i32(at), qr, kr)
        ctx.kv4_write(cache, kr, v.to(t), i32([0, 1, 2]), i32(at))
        now = [n + 1 for n in at]
        o = torch.empty(2, 1, H, hd, dtype=t, device="cuda")
        ctx.kv4_attention(cache, qr[:, None], i32(now), o, work)
        ctx.sync()
        want, tol = cached_reference(cache, table, qr[:, None], now, 0, hd ** -0.5, None)
        within(o, want, tol)


def test_captured_decode_step_replays_on_another_stream(ctx):
    """One captured step (norm and rotation, write, attention) replayed with new contents of the same tensors, on a
    stream of its own; the eager call gives the same bits."""
    from moe_stream_b200.engine import Context
    H, kv, hd, t = 16, 2, 64, torch.bfloat16
    lens0 = [50, 200, 9]
    cache, _, table = new_cache([n + 4 for n in lens0], 16, kv, hd, seed=3, fill=0xFF)
    fill_cache(ctx, cache, lens0, 1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    c2 = Context(0, stream=stream)
    _, q, k, qw, kw, cos, sin, _ = rope_inputs(3, H, kv, hd, hd, True, torch.float32, seed=2)
    cos, sin = cos.repeat(8, 1), sin.repeat(8, 1)                # positions up to 8 * 43
    v = torch.randn(3, kv, hd, device="cuda", generator=gen(1)).to(t)
    pos, lens = i32(lens0), i32([n + 1 for n in lens0])
    qr, kr = torch.empty(3, H, hd, dtype=t, device="cuda"), torch.empty(3, kv, hd, dtype=t, device="cuda")
    o, cu = torch.empty(3, 1, H, hd, dtype=t, device="cuda"), i32([0, 1, 2, 3])
    n = c2.kv4_attention_workspace_bytes(cache, 3, 1, H)
    work, other = (torch.empty(n, dtype=torch.uint8, device="cuda") for _ in range(2))

    def step(c, w, out):
        c.qk_norm_rope(q, k, qw, kw, 1e-6, cos, sin, pos, qr, kr)
        c.kv4_write(cache, kr, v, cu, pos)
        c.kv4_attention(cache, qr[:, None], lens, out, w)

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        step(c2, work, o)
    for s in range(3):
        q.copy_(torch.randn(q.shape, device="cuda", generator=gen(50 + s)))
        k.copy_(torch.randn(k.shape, device="cuda", generator=gen(60 + s)))
        v.copy_(torch.randn(v.shape, device="cuda", generator=gen(70 + s)))
        pos.copy_(i32([x + s for x in lens0]))
        lens.copy_(i32([x + s + 1 for x in lens0]))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        c2.sync()
        now = [x + s + 1 for x in lens0]
        want, tol = cached_reference(cache, table, qr[:, None], now, 0, hd ** -0.5, None)
        within(o, want, tol)
        eager = torch.empty_like(o)
        step(ctx, other, eager)
        ctx.sync()
        assert torch.equal(o, eager)
    c2.close()
