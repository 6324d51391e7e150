"""GPU tests of the attention operators at edges of their walks, against the 64-bit forms and tolerances of
test_gpu_attn_ops."""
import numpy as np
import pytest

from . import attn_ref as R
from . import test_gpu_attn_ops as G
from .test_gpu_attn_ops import ctx  # noqa: F401  (fixture)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompt_attention_ends_of_short_walks_beside_other_work(ctx, hd):
    """Walks of 1 to 6 key tiles, many times, while another stream's kernels come and go on the same SMs: every softmax
    warp's last waits pass, wherever the last products stand."""
    from moe_stream_b200.engine import Context
    sets = []
    for tiles in range(1, 7):
        q, k, v, cq, ck, both, _ = G.prompt_case([90], [128 * tiles - 100], 16, 2, hd, torch.bfloat16, seed=tiles, behind=0)
        first = torch.empty_like(q)
        ctx.prompt_attention(q, k, v, cq, ck, first)
        ctx.sync()
        G.within(first, *G.prompt_reference(q, k, v, [90], both, 0, hd ** -0.5, None))
        sets.append(((q, k, v, cq, ck), first, [torch.empty_like(q) for _ in range(20)]))
    side = torch.cuda.Stream()
    c2 = Context(0, stream=side)
    x = torch.randn(1 << 16, device="cuda")
    torch.cuda.synchronize()
    for r in range(20):
        with torch.cuda.stream(side):
            for n in (1, 3, 16):
                x[:n << 12].mul_(1.0)
        c2.prompt_attention(*sets[r % 6][0], torch.empty_like(sets[r % 6][1]))
        for args, _, outs in sets:
            ctx.prompt_attention(*args, outs[r])
    ctx.sync()
    c2.sync()
    for _, first, outs in sets:
        assert all(torch.equal(o, first) for o in outs)
    c2.close()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("entry", [-1, -2, -3, -2 ** 31, 2 ** 31 - 1])
def test_kv4_attention_reports_every_bad_page_number(ctx, page, entry):
    """The entry of a page that is attended; the result is the attention of the tokens that are there (half a step of bf16, and
    2^-11 of p and of v and the scores' errors, together below 2^-8 of A)."""
    from moe_stream_b200._lib import MsError
    case = ([4 * page], 1, page, 8, 1, 64, 0, False, "bfloat16")
    cache, table, q, lens, out, work, _, _ = G.cached_case(ctx, case, poison=False)
    raw = cache.pages.cpu().numpy()
    k, v = (torch.from_numpy(x).cuda() for x in R.cache_values(raw, table, 0, 4 * page, page, 1, 64)[:2])
    keep = [j for j in range(4 * page) if j // page != 2]
    cache.block_table[0, 2] = entry
    ctx.kv4_attention(cache, q, lens, out, work)
    with pytest.raises(MsError) as e:
        ctx.sync()
    assert e.value.status == 11
    want, A = R.attention(q[0], k[keep], v[keep], torch.tensor([4 * page], device="cuda"), 0, 0.125, None)
    G.within(out[0], want, 2.0 ** -8 * want.abs() + 2.0 ** -8 * A)


# ---------------------------------------------------------------- offsets that are not the offsets of packed sequences

def reported(ctx):
    from moe_stream_b200._lib import MsError
    with pytest.raises(MsError) as e:
        ctx.sync()
    assert e.value.status == 11
    ctx.sync()


def bad_offsets(n, total, how):
    """Offsets of n sequences of `total` rows, bad in one place."""
    cu = [i * total // n for i in range(n + 1)]
    if how == "descends":
        cu[n // 2] = cu[n // 2 + 1] + 3
    elif how == "negative":
        cu[0] = -2
    elif how == "behind":
        cu[n] = total + 1
    else:                                                        # a sequence in the middle begins before its predecessor
        cu[n // 2 + 1] = max(0, cu[n // 2] - 5)
    return cu


@pytest.mark.parametrize("n", [2, 40, 3000])
@pytest.mark.parametrize("how", ["descends", "negative", "behind", "overlaps"])
def test_kv4_rows_report_bad_offsets(ctx, n, how):
    total = 2 * n + 10
    cache, raw, table = G.new_cache([32] * n, 16, 1, 64, seed=n)
    cu, start = G.i32(bad_offsets(n, total, how)), G.i32([0] * n)
    k = torch.randn(total, 1, 64, device="cuda", generator=G.gen(1)).half()
    ctx.kv4_write(cache, k, k, cu, start)
    reported(ctx)
    nobody = sorted(set(range(raw.shape[0])) - set(table.reshape(-1).tolist()))
    assert np.array_equal(cache.pages.cpu().numpy()[nobody], raw[nobody])
    ctx.kv4_read(cache, cu, start, torch.empty_like(k), torch.empty_like(k))
    reported(ctx)
    good = G.i32([i * total // n for i in range(n + 1)])
    ctx.kv4_write(cache, k, k, good, start)
    ctx.kv4_read(cache, good, start, torch.empty_like(k), torch.empty_like(k))
    ctx.sync()


@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("n", [2, 40, 3000])
@pytest.mark.parametrize("how", ["descends", "negative", "behind", "overlaps"])
def test_prompt_attention_reports_bad_offsets(ctx, n, how, hd):
    total = 2 * n + 10
    q = torch.randn(total, 4, hd, device="cuda", generator=G.gen(2)).half()
    k = torch.randn(total, 2, hd, device="cuda", generator=G.gen(3)).half()
    good, bad, out = G.i32([i * total // n for i in range(n + 1)]), G.i32(bad_offsets(n, total, how)), torch.empty_like(q)
    for cq, ck in ((bad, good), (good, bad)):
        ctx.prompt_attention(q, k, k, cq, ck, out)
        reported(ctx)
    ctx.prompt_attention(q, k, k, good, good, out)
    ctx.sync()


def test_rows_in_front_of_the_first_sequence_are_left(ctx):
    """Offsets that begin behind 0 are no error: the rows in front of them are nobody's."""
    cache, raw, table = G.new_cache([20], 16, 2, 64, seed=1)
    k = torch.randn(30, 2, 64, device="cuda", generator=G.gen(1)).half()
    ctx.kv4_write(cache, k, k, G.i32([10, 30]), G.i32([0]))
    back = torch.full_like(k, 7.0)
    ctx.kv4_read(cache, G.i32([10, 30]), G.i32([0]), back, torch.empty_like(k))
    q = torch.randn(30, 4, 64, device="cuda", generator=G.gen(2)).half()
    out, want = torch.full_like(q, 7.0), torch.empty_like(q[10:])
    ctx.prompt_attention(q, k, k, G.i32([10, 30]), G.i32([10, 30]), out)
    ctx.prompt_attention(q[10:], k[10:], k[10:], G.i32([0, 20]), G.i32([0, 20]), want)
    ctx.sync()
    assert (back[:10] == 7.0).all() and (back[10:] != 7.0).any()
    assert (out[:10] == 7.0).all() and torch.equal(out[10:], want)


# ---------------------------------------------------------------- one large score in front of many small ones

def spike_rows(n, hd, seed):
    """K and V rows of one kv head: key 0 is all ones with v = 0, the others are zeros with v between 1 and 1.25."""
    g = G.gen(seed)
    k = torch.zeros(n, 1, hd, device="cuda")
    k[0] = 1.0
    v = 1 + 0.25 * torch.rand(n, 1, hd, device="cuda", generator=g)
    v[0] = 0
    return k, v


def spike_queries(n, hd, drop, t):
    """One query of n heads: the probability of key 0 is 2^drop[head] times that of any other key."""
    q = torch.tensor(drop, device="cuda")[None, :, None] / (np.log2(np.e) * hd ** 0.5)
    return q.expand(1, n, hd).contiguous().to(t)


DROPS = [0.0, 14.5, 20.5, 24.9, 25.5, 26.0, 27.5, 29.0]            # 2^-25 and below round to 0 in f16


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("t", ["float16", "bfloat16"])
def test_kv4_attention_large_score_and_flat_tail(ctx, hd, t):
    """All that the output has comes from keys with probabilities of 2^-14.5 .. 2^-29 of the largest.  512 sequences that
    share one's pages, so that a warp takes many keys behind the large one.  Besides the roundings of G.cached_reference, a
    probability is off by half an f16 subnormal, 2^-25 where the largest is 2^7 or more: 2^-32 of it for each key."""
    from moe_stream_b200.engine import KV4Cache
    t, n, seqs = getattr(torch, t), 4000, 512
    one, _, table = G.new_cache([n], 16, 1, hd, seed=1)
    k, v = spike_rows(n, hd, 2)
    ctx.kv4_write(one, k, v, G.i32([0, n]), G.i32([0]))
    ctx.sync()
    cache = KV4Cache(one.pages, one.block_table.expand(seqs, -1).contiguous(), 1, hd, 16)
    q = spike_queries(len(DROPS), hd, DROPS, t)[None].expand(seqs, -1, -1, -1).contiguous()
    out = torch.empty_like(q)
    work = torch.empty(ctx.kv4_attention_workspace_bytes(cache, seqs, 1, len(DROPS)), dtype=torch.uint8, device="cuda")
    ctx.kv4_attention(cache, q, G.i32([n] * seqs), out, work)
    ctx.sync()
    want, tol = G.cached_reference(one, table, q[:1], [n], 0, hd ** -0.5, None)
    G.within(out, want.expand_as(out), (tol + n * 2.0 ** -32 * 1.25).expand_as(out))


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("t", ["float16", "bfloat16"])
def test_prompt_attention_large_score_and_flat_tail(ctx, hd, t):
    """The same for one query behind 4,000 keys (each head a drop): f16 probabilities are off by 2^-32 of the largest for
    each key, bf16 ones by nothing besides their rounding."""
    t, n, H = getattr(torch, t), 4000, len(DROPS)
    k, v = (x.to(t) for x in spike_rows(n, hd, 3))
    q = spike_queries(H, hd, DROPS, t)
    out = torch.empty_like(q)
    cq, ck = G.i32([0, 1]), G.i32([0, n])
    ctx.prompt_attention(q, k, v, cq, ck, out)
    ctx.sync()
    want, tol = G.prompt_reference(q, k, v, [1], [n], 0, hd ** -0.5, None)
    G.within(out, want, tol + n * 2.0 ** -32 * 1.25)


# ---------------------------------------------------------------- sinks that are no numbers

@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("longest", [40, 9000])                      # one block's part of a job, and joined parts
def test_a_nan_sink_reaches_its_head_alone(ctx, hd, longest):
    """A NaN sink makes its head's rows NaN, where they have keys; the other heads, with finite and infinite sinks, are as
    without it."""
    H = 8
    case = ([longest, 0, 3], 4, 16, H, 2, hd, 0, False, "float16")
    cache, table, q, lens, out, work, _, _ = G.cached_case(ctx, case, poison=True)
    pq, pk, pv, cq, ck, _, _ = G.prompt_case([70, 40], [0, 9], H, 2, hd, torch.float16)
    sk = torch.randn(H, device="cuda", generator=G.gen(9))
    sk[1], sk[6] = float("inf"), float("-inf")
    bad = sk.clone()
    bad[3] = float("nan")
    nan, pn, pw = torch.empty_like(out), torch.empty_like(pq), torch.empty_like(pq)
    ctx.kv4_attention(cache, q, lens, out, work, sinks=sk)
    ctx.kv4_attention(cache, q, lens, nan, work, sinks=bad)
    ctx.prompt_attention(pq, pk, pv, cq, ck, pw, sinks=sk)
    ctx.prompt_attention(pq, pk, pv, cq, ck, pn, sinks=bad)
    ctx.sync()
    keep = [h for h in range(H) if h != 3]
    assert torch.equal(nan[:, :, keep], out[:, :, keep]) and torch.equal(pn[:110, keep], pw[:110, keep])
    assert torch.isnan(nan[0, :, 3]).all() and torch.isnan(nan[2, 1:, 3]).all() and torch.isnan(pn[:110, 3]).all()
    assert (nan[1, :, 3] == 0).all() and (nan[2, 0, 3] == 0).all()   # queries without keys
    assert (out[:, :, 1] == 0).all() and (pw[:110, 1] == 0).all()
