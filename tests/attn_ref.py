"""Plain restatements of the attention operators for the tests: the 4-bit cache's layout byte by byte
(numpy), and rotation and attention in 64 bits (torch, on any device)."""
import numpy as np
import torch


def quantise(x):
    """x [..., 32] f32 -> (codes, d, o) in the IEEE f32 operations of the definition."""
    x = np.where(np.isnan(x), np.float32(0), np.clip(x.astype(np.float32), -16384, 16384)).astype(np.float32)
    lo, hi = x.min(-1), x.max(-1)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        d = ((hi - lo) / np.float32(15)).astype(np.float16)
        df = d.astype(np.float32)
        o = (lo - np.float32(16) * df).astype(np.float16)
        c = np.rint((x - o.astype(np.float32)[..., None]) / df[..., None]) - np.float32(16)
    c = np.where(df[..., None] > 0, c, 0)
    return np.clip(c, 0, 15).astype(np.int64), d, o


def block_bytes(hd):
    return 20 * hd


def _k_at(hd, tok, dim):
    """(byte, shift) of a K code and byte of its scales in a block."""
    G = hd // 32
    w, t, n, h = dim // 32, dim % 32 // 8, dim % 8 // 2, dim % 2
    return (tok * 4 * G + t * G + w) * 4 + (4 * n + 16 * h) // 8, (4 * n + 16 * h) % 8, 8 * hd + (tok * G + w) * 4


def _v_at(hd, tok, dim):
    G, pair, par, C = hd // 32, tok // 2, tok % 2, dim // 16
    C = C ^ (pair & 2) if hd == 64 else C ^ ((pair & 3) << 1)
    bit = 4 * (dim % 4)
    u16 = (pair * (hd // 16) + C) * 8 + dim % 16 // 4 * 2 + par
    return 10 * hd + u16 * 2 + bit // 8, bit % 8, 18 * hd + (pair * G + dim // 32) * 8 + 2 * par


def put_token(pages, table, seq, pos, page_tokens, kv_heads, hd, k, v):
    """Store one token's rows k / v [kv_heads][hd] in pages (numpy uint8 [n_pages][kv_heads][blocks][20 hd])."""
    page = table[seq, pos // page_tokens]
    tok, b = pos % 16, pos % page_tokens // 16
    for h in range(kv_heads):
        blk = pages[page, h, b]
        for x, at, second in ((k[h], _k_at, 2), (v[h], _v_at, 4)):
            c, d, o = quantise(x.reshape(-1, 32))
            for dim in range(hd):
                byte, sh, sc = at(hd, tok, dim)
                blk[byte] = (blk[byte] & (0xF0 if sh == 0 else 0x0F)) | (int(c[dim // 32, dim % 32]) << sh)
                if dim % 32 == 0:
                    blk[sc:sc + 2] = np.frombuffer(d[dim // 32].tobytes(), np.uint8)
                    blk[sc + second:sc + second + 2] = np.frombuffer(o[dim // 32].tobytes(), np.uint8)


def cache_values(pages, table, seq, n, page_tokens, kv_heads, hd):
    """(k, v, d_k, o_k, d_v, o_v) f64 [n][kv_heads][hd] of a sequence's first n tokens."""
    pos = np.arange(n)
    page = np.asarray(table)[seq, pos // page_tokens]
    blk = pages[page, :, pos % page_tokens // 16]               # [n][kv_heads][20 hd]
    out = []
    for at, second in ((_k_at, 2), (_v_at, 4)):
        byte, sh, sc = (np.array([[at(hd, t, i)[j] for i in range(hd)] for t in range(16)]) for j in range(3))
        tok = pos % 16
        take = lambda idx: np.take_along_axis(blk, np.broadcast_to(idx[tok][:, None], blk.shape[:2] + (hd,)), 2)
        code = (take(byte) >> sh[tok][:, None]) & 15
        f16 = lambda idx: (take(idx).astype(np.uint16) | (take(idx + 1).astype(np.uint16) << 8)).view(np.float16)
        d, o = f16(sc).astype(np.float64), f16(sc + second).astype(np.float64)
        out.append((o + d * (16 + code), d, o))
    (k, dk, ok), (v, dv, ov) = out
    return k, v, dk, ok, dv, ov


def rope(x, w, eps, cos, sin, pos, interleaved):
    """RMSNorm and rotation of x [tokens][heads][hd] in f64; also |a| + |b| of each value's pair."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    half = cos.shape[1]
    c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
    ia = torch.arange(half, device=x.device) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else half)
    a, b = x[..., ia], x[..., ib]
    y, size = x.clone(), x.abs()
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = a.abs() + b.abs()
    return y, size


def attention(q, k, v, place, window, scale, sinks):
    """One sequence in f64: q [n][H][hd], k / v [m][kv][hd], place [n] each query's key index.  Returns
    (out, sum p |v| / sum p), rows without keys zero."""
    n, H, hd = q.shape
    rep = H // k.shape[1]
    k, v = k.double().repeat_interleave(rep, 1), v.double().repeat_interleave(rep, 1)
    s = torch.einsum("nhd,mhd->hnm", q.double(), k) * scale
    j = torch.arange(k.shape[0], device=q.device)
    ok = j <= place[:, None]
    if window > 0:
        ok &= j > place[:, None] - window
    s = s.masked_fill(~ok, float("-inf"))
    if sinks is not None:
        s = torch.cat((s, sinks.double().view(H, 1, 1).expand(H, n, 1)), 2)
    if s.shape[2] == 0:
        z = torch.zeros(n, H, hd, dtype=torch.float64, device=q.device)
        return z, z
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    den = p.sum(-1, keepdim=True)
    p = (p / torch.where(den > 0, den, 1.0))[..., :k.shape[0]]
    return torch.einsum("hnm,mhd->nhd", p, v), torch.einsum("hnm,mhd->nhd", p, v.abs())
