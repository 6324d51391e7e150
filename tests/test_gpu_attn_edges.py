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
