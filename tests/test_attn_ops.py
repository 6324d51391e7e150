"""CPU checks of the attention operators: what their entry points refuse (a null context runs the checks alone),
and the 4-bit cache's layout."""
import ctypes as C

import numpy as np
import pytest

from moe_stream_b200 import _lib

from . import attn_ref as R

INVALID, QTYPE, SHAPE = 1, 6, 7
P = 4096   # stands for a device pointer; nothing is launched


@pytest.fixture(scope="module")
def L():
    from moe_stream_b200 import build
    build.build()
    return _lib.lib()


def make(cls, **kw):
    a = cls()
    for k, v in kw.items():
        setattr(a, k, v)
    return a


ROPE = dict(n_tokens=3, heads=8, kv_heads=2, head_dim=128, rot_dim=64, in_type=0, out_type=30, eps=1e-6, max_pos=10, q=P,
            k=P, q_stride=1024, k_stride=256, q_norm=P, k_norm=P, cos_t=P, sin_t=P, pos=P, q_out=2 * P, k_out=2 * P,
            q_out_stride=1024, k_out_stride=256)
ROPE_BIG = dict(q_stride=1 << 40, k_stride=1 << 40, q_out_stride=1 << 40, k_out_stride=1 << 40)
PROMPT = dict(n_seqs=2, heads=8, kv_heads=2, head_dim=64, type=30, total_q=10, total_k=20, q=P, k=P, v=P, q_stride=512,
              k_stride=128, v_stride=128, cu_q=P, cu_k=P, out=2 * P, out_stride=512)
CACHE = dict(kv_heads=2, head_dim=128, page_tokens=16, n_pages=5, pages=P, block_table=P, n_seqs=2, max_pages=3)
ROWS = dict(type=30, total=7, cu=P, start=P, k=P, v=P, k_stride=256, v_stride=256)
ATTN = dict(n_query=1, heads=8, type=1, q=P, lens=P, out=2 * P, work=P, work_bytes=1 << 30)


@pytest.mark.parametrize("change,status", [
    ({}, INVALID), (dict(n_tokens=0, q=None, pos=None), INVALID),     # fine but for the context
    (dict(n_tokens=-1), SHAPE), (dict(heads=0), SHAPE), (dict(kv_heads=0), SHAPE), (dict(max_pos=0), SHAPE),
    (dict(head_dim=127), SHAPE), (dict(head_dim=514, q_stride=8192, k_stride=8192), SHAPE), (dict(rot_dim=130), SHAPE),
    (dict(rot_dim=0), SHAPE), (dict(rot_dim=7), SHAPE), (dict(in_type=8), QTYPE), (dict(out_type=2), QTYPE),
    (dict(q_stride=1023), SHAPE), (dict(k_out_stride=255), SHAPE), (dict(n_tokens=1 << 30), SHAPE),
    (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID), (dict(q_norm=None), INVALID), (dict(pos=None), INVALID),
    (dict(q_out=P), INVALID),                                         # in place needs the input's type
], ids=str)
def test_rope_refusals(L, change, status):
    assert L.ms_qk_norm_rope(None, C.byref(make(_lib.QkRope, **{**ROPE, **change}))) == status
    assert L.ms_qk_norm_rope(None, None) == INVALID


@pytest.mark.parametrize("change,status", [
    ({}, INVALID), (dict(total_q=0, q=None, out=None), INVALID),
    (dict(n_seqs=-1), SHAPE), (dict(total_k=-1), SHAPE), (dict(heads=9), SHAPE), (dict(heads=0), SHAPE),
    (dict(heads=258, q_stride=1 << 15, out_stride=1 << 15), SHAPE), (dict(head_dim=96, q_stride=4096), SHAPE),
    (dict(type=0), QTYPE), (dict(type=8), QTYPE), (dict(q_stride=504), SHAPE), (dict(v_stride=132), SHAPE),
    (dict(k=P + 8), SHAPE), (dict(out=P + 2), SHAPE), (dict(scale=-1.0), INVALID), (dict(scale=float("inf")), INVALID),
    (dict(cu_q=None), INVALID), (dict(v=None), INVALID), (dict(out=P), INVALID), (dict(total_q=1 << 30), SHAPE),
], ids=str)
def test_prompt_refusals(L, change, status):
    assert L.ms_prompt_attention(None, C.byref(make(_lib.PromptAttn, **{**PROMPT, **change}))) == status


@pytest.mark.parametrize("change", [
    dict(q=P + 1), dict(k_out=P + 1), dict(in_type=1, k=P + 1), dict(out_type=0, q_out=P + 2), dict(q_norm=P + 2), dict(cos_t=P + 1),
    dict(sin_t=P + 2), dict(pos=P + 2), dict(n_tokens=1, heads=65537, **ROPE_BIG), dict(n_tokens=1, kv_heads=1 << 24, **ROPE_BIG),
], ids=str)
def test_rope_addresses_between_elements_and_row_offsets(L, change):
    assert L.ms_qk_norm_rope(None, C.byref(make(_lib.QkRope, **{**ROPE, **change}))) == SHAPE
    fine = {k: v // 4 * 4 if k not in ("heads", "kv_heads") else 65536 for k, v in change.items() if not k.endswith("_type")}
    assert L.ms_qk_norm_rope(None, C.byref(make(_lib.QkRope, **{**ROPE, **fine}))) == INVALID


@pytest.mark.parametrize("change", [dict(cu_q=P + 2), dict(cu_k=P + 1), dict(sinks=P + 2),
                                    dict(heads=131072, kv_heads=65536, q_stride=1 << 30, out_stride=1 << 30, k_stride=1 << 30, v_stride=1 << 30)], ids=str)
def test_prompt_addresses_between_elements_and_row_offsets(L, change):
    assert L.ms_prompt_attention(None, C.byref(make(_lib.PromptAttn, **{**PROMPT, **change}))) == SHAPE


@pytest.mark.parametrize("name", ["block_table", "cu", "start", "lens", "sinks"])
def test_cache_addresses_between_elements(L, name):
    def calls(at):
        c = make(_lib.Kv4CacheArgs, **{**CACHE, **({name: at} if name in CACHE else {})})
        r = make(_lib.Kv4Rows, **{**ROWS, **({name: at} if name in ROWS else {})})
        a = make(_lib.Kv4Attn, **{**ATTN, **({name: at} if name in ("lens", "sinks") else {})})
        rows = [L.ms_kv4_write(None, C.byref(c), C.byref(r)), L.ms_kv4_read(None, C.byref(c), C.byref(r))]
        attn = [L.ms_kv4_attention(None, C.byref(c), C.byref(a))]
        return rows + attn if name in CACHE else rows if name in ROWS else attn
    assert set(calls(P + 2)) == {SHAPE}
    assert set(calls(P + 4)) == {INVALID}                             # fine but for the context


CACHE_BAD = [(dict(kv_heads=0), SHAPE), (dict(kv_heads=70000), SHAPE), (dict(head_dim=96), SHAPE), (dict(page_tokens=8), SHAPE), (dict(page_tokens=48), SHAPE),
             (dict(page_tokens=2048), SHAPE), (dict(pages=P + 4), SHAPE), (dict(pages=None), INVALID),
             (dict(block_table=None), INVALID), (dict(max_pages=1 << 28), SHAPE), (dict(n_seqs=-1), SHAPE)]


@pytest.mark.parametrize("cache,rows,status", [
    ({}, {}, INVALID), ({}, dict(total=0, k=None), INVALID),
    *[(c, {}, s) for c, s in CACHE_BAD],
    ({}, dict(total=-1), SHAPE), ({}, dict(total=1 << 30), SHAPE), ({}, dict(type=8), QTYPE), ({}, dict(k_stride=248), SHAPE),
    ({}, dict(v_stride=260), SHAPE), ({}, dict(k=P + 8), SHAPE), ({}, dict(cu=None), INVALID), ({}, dict(v=None), INVALID),
], ids=str)
def test_cache_row_refusals(L, cache, rows, status):
    c, r = make(_lib.Kv4CacheArgs, **{**CACHE, **cache}), make(_lib.Kv4Rows, **{**ROWS, **rows})
    assert L.ms_kv4_write(None, C.byref(c), C.byref(r)) == status
    assert L.ms_kv4_read(None, C.byref(c), C.byref(r)) == status


@pytest.mark.parametrize("cache,attn,status", [
    ({}, {}, INVALID), *[(c, {}, s) for c, s in CACHE_BAD],
    ({}, dict(n_query=0), SHAPE), ({}, dict(heads=9), SHAPE), ({}, dict(n_query=33), SHAPE), ({}, dict(type=0), QTYPE),
    (dict(n_seqs=70000), {}, SHAPE), (dict(n_seqs=60000, max_pages=1 << 20), {}, SHAPE),
    ({}, dict(scale=float("nan")), INVALID), ({}, dict(q=P + 2), SHAPE), ({}, dict(work=P + 8), SHAPE),
    ({}, dict(lens=None), INVALID), ({}, dict(work=None), INVALID), ({}, dict(out=P), INVALID),
], ids=str)
def test_cached_attention_refusals(L, cache, attn, status):
    c, a = make(_lib.Kv4CacheArgs, **{**CACHE, **cache}), make(_lib.Kv4Attn, **{**ATTN, **attn})
    assert L.ms_kv4_attention(None, C.byref(c), C.byref(a)) == status


def test_page_bytes(L):
    n = C.c_size_t()
    for kv, hd, page in ((1, 64, 16), (4, 128, 64), (2, 256, 1024)):
        assert L.ms_kv4_page_bytes(kv, hd, page, C.byref(n)) == 0
        assert n.value == kv * page // 16 * R.block_bytes(hd) == kv * page * hd * 5 // 4
    for kv, hd, page in ((0, 64, 16), (1, 32, 16), (1, 64, 17)):
        assert L.ms_kv4_page_bytes(kv, hd, page, C.byref(n)) == SHAPE
    assert L.ms_kv4_page_bytes(1, 64, 16, None) == INVALID


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_layout_covers_a_block_once(hd):
    """Every code has a nibble and every scale its bytes; together they fill the block."""
    seen = np.zeros(R.block_bytes(hd) * 2, np.int64)             # nibbles
    for tok in range(16):
        for dim in range(hd):
            for at, second in ((R._k_at, 2), (R._v_at, 4)):
                byte, sh, sc = at(hd, tok, dim)
                seen[2 * byte + sh // 4] += 1
                if dim % 32 == 0:
                    seen[2 * sc:2 * sc + 4] += 1
                    seen[2 * (sc + second):2 * (sc + second) + 4] += 1
    assert (seen == 1).all()


def test_quantised_values_are_near(hd=128):
    r = np.random.default_rng(0)
    x = (r.standard_normal((64, 32)) * r.uniform(0.01, 50, (64, 1))).astype(np.float32)
    c, d, o = R.quantise(x)
    d, o = d.astype(np.float64)[:, None], o.astype(np.float64)[:, None]
    err = np.abs(o + d * (16 + c) - x)
    assert (err <= d * (0.5 + 31 * 2.0 ** -11) + np.abs(o) * 2.0 ** -11).all()


# ---------------------------------------------------------------- the binding: tensors on the CPU, no context behind it

class Calls:
    """The calls of a context without a device, with tensors that fit; a change replaces one."""

    def __init__(self):
        import torch
        from moe_stream_b200 import Context, KV4Cache
        self.torch = torch
        self.ctx = object.__new__(Context)
        self.ctx.h, self.ctx.device = None, -1                        # CPU tensors are on device -1
        bf, i32 = torch.bfloat16, torch.int32
        z = torch.zeros
        cache = KV4Cache(z(5 * KV4Cache.page_bytes(2, 64, 16), dtype=torch.uint8), z(3, 4, dtype=i32), 2, 64, 16)
        rows = dict(cache=cache, k=z(7, 2, 64, dtype=bf), v=z(7, 2, 64, dtype=bf), cu=z(4, dtype=i32), start=z(3, dtype=i32))
        self.args = {
            "qk_norm_rope": dict(q=z(5, 8, 64), k=z(5, 2, 64), q_norm=z(64), k_norm=z(64), eps=1e-6, cos=z(9, 32), sin=z(9, 32),
                                 pos=z(5, dtype=i32), q_out=z(5, 8, 64, dtype=bf), k_out=z(5, 2, 64, dtype=bf)),
            "prompt_attention": dict(q=z(6, 8, 64, dtype=bf), k=z(9, 2, 64, dtype=bf), v=z(9, 2, 64, dtype=bf), cu_q=z(4, dtype=i32),
                                     cu_k=z(4, dtype=i32), out=z(6, 8, 64, dtype=bf), window=3, sinks=z(8), scale=0.5),
            "kv4_write": rows, "kv4_read": dict(rows),
            "kv4_attention": dict(cache=cache, q=z(3, 1, 8, 64, dtype=bf), lens=z(3, dtype=i32), out=z(3, 1, 8, 64, dtype=bf),
                                  work=z(64, dtype=torch.uint8), window=0, sinks=None, scale=0.0),
        }

    def call(self, name, **change):
        return getattr(self.ctx, name)(**{**self.args[name], **change})


@pytest.fixture(scope="module")
def calls(L):
    return Calls()


@pytest.mark.parametrize("name", ["qk_norm_rope", "prompt_attention", "kv4_write", "kv4_read", "kv4_attention"])
def test_binding_reaches_the_library(calls, name):
    with pytest.raises(_lib.MsError) as e:                            # what fits is refused for want of a context alone
        calls.call(name)
    assert e.value.status == INVALID
    calls.ctx.device = 0                                              # and for another device before that
    with pytest.raises(ValueError, match="the context on cuda:0"):
        calls.call(name)
    calls.ctx.device = -1


@pytest.mark.parametrize("name,arg,make", [
    ("qk_norm_rope", "q", lambda t: t[:, :, :63]), ("qk_norm_rope", "q", lambda t: t[0]), ("qk_norm_rope", "k", lambda t: t.half()),
    ("qk_norm_rope", "k", lambda t: t[:4]), ("qk_norm_rope", "q_norm", lambda t: t[:63]), ("qk_norm_rope", "k_norm", lambda t: t.double()),
    ("qk_norm_rope", "cos", lambda t: t[:8]), ("qk_norm_rope", "sin", lambda t: t.t()), ("qk_norm_rope", "pos", lambda t: t.long()),
    ("qk_norm_rope", "pos", lambda t: t[:4]), ("qk_norm_rope", "q_out", lambda t: t.float()), ("qk_norm_rope", "k_out", lambda t: t[:, :1]),
    ("qk_norm_rope", "q", lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)),
    ("prompt_attention", "k", lambda t: t[:8]), ("prompt_attention", "v", lambda t: t.half()), ("prompt_attention", "out", lambda t: t[:5]),
    ("prompt_attention", "cu_q", lambda t: t[:3]), ("prompt_attention", "cu_k", lambda t: t.long()),
    ("prompt_attention", "sinks", lambda t: t.bfloat16()), ("prompt_attention", "sinks", lambda t: t[::2]),
    ("prompt_attention", "window", lambda w: 1 << 40), ("prompt_attention", "q", lambda t: t.transpose(1, 2)),
    ("kv4_write", "k", lambda t: t[:6]), ("kv4_write", "v", lambda t: t.float()), ("kv4_read", "cu", lambda t: t[:3]),
    ("kv4_read", "start", lambda t: t.float()), ("kv4_read", "k", lambda t: t.reshape(7, 128)),
    ("kv4_attention", "q", lambda t: t[:2]), ("kv4_attention", "out", lambda t: t.half()), ("kv4_attention", "lens", lambda t: t[:2]),
    ("kv4_attention", "q", lambda t: t[:, 0]), ("kv4_attention", "out", lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)),
])
def test_binding_refuses_what_does_not_fit(calls, name, arg, make):
    with pytest.raises(ValueError):
        calls.call(name, **{arg: make(calls.args[name][arg])})


@pytest.mark.parametrize("name,arg,value", [("qk_norm_rope", "q", None), ("prompt_attention", "cu_q", [0, 1]), ("kv4_write", "k", 4096),
                                            ("kv4_attention", "work", "x"), ("prompt_attention", "scale", "y"), ("kv4_attention", "window", 1.5)])
def test_binding_refuses_other_types(calls, name, arg, value):
    with pytest.raises(TypeError):
        calls.call(name, **{arg: value})


def test_binding_takes_strided_rows_and_one_token(calls):
    t = calls.torch
    fused = t.zeros(5, 12 * 64)                                       # the fused projection's rows
    q, k = fused[:, :512].view(5, 8, 64), fused[:, 512:640].view(5, 2, 64)
    one = dict(q=q[:1], k=k[:1], pos=calls.args["qk_norm_rope"]["pos"][:1], q_out=t.zeros(1, 8, 64), k_out=t.zeros(1, 2, 64))
    for change in (dict(q=q, k=k), one, dict(q_norm=None, k_norm=None), dict(interleaved=True)):
        with pytest.raises(_lib.MsError) as e:
            calls.call("qk_norm_rope", **change)
        assert e.value.status == INVALID


def test_binding_refuses_what_is_neither_true_nor_false(calls):
    class Neither:
        def __bool__(self):
            raise RuntimeError("neither")
    with pytest.raises(RuntimeError, match="neither"):
        calls.call("qk_norm_rope", interleaved=Neither())
