"""Plain implementations of the paged 4-bit KV cache's operators (numpy, from their definitions)."""
import numpy as np

F = np.float32


def to_bf16(x):
    """Round to nearest even, as bit patterns."""
    u = np.ascontiguousarray(x, F).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(b):
    return (np.ascontiguousarray(b, np.uint16).astype(np.uint32) << 16).view(F)


def codec(x):
    """The value every element of f32 [..., 64 n] is held as: (nibble, scale, bias) of its group of 64, in f32 steps."""
    x = np.ascontiguousarray(x, F)
    g = x.reshape(-1, 64)
    lo, hi = g.min(1), g.max(1)
    hi = np.where(hi == lo, lo + F(1), hi)
    scale = (hi - lo) / F(15)
    t = (g - lo[:, None]) * (F(1) / scale)[:, None] + F(0.5)
    n = np.clip(np.trunc(t), 0, 15).astype(F)

    def rounded(v):  # the packer's f32 -> bf16: up when bit 15 is set together with bit 0 or bit 16
        u = v.view(np.uint32)
        up = (u >> 15) & ((u & 0x7FFF) | (u >> 16)) & 1
        return (((u + (up << 16)) >> 16) << 16).view(F)

    return (n * rounded(scale)[:, None] + rounded(lo)[:, None]).reshape(x.shape)


def rotate_f32(x, cs, interleaved):
    """x f32 [T, H, dim], cs f32 [T, rotary] (cosines, sines): every product and sum rounded to f32."""
    r = cs.shape[-1]
    c, s = cs[:, None, :r // 2], cs[:, None, r // 2:]
    ia = np.arange(0, r, 2) if interleaved else np.arange(r // 2)
    ib = ia + 1 if interleaved else ia + r // 2
    y = np.array(x, F)
    a, b = y[..., ia].copy(), y[..., ib].copy()
    y[..., ia] = a * c - b * s
    y[..., ib] = a * s + b * c
    return y


def attention(q, k, v, lens, q_lens, window, scale):
    """q f64 [rows, heads, dim]; k, v of the sequences back to back [sum lens, kv_heads, dim] -> result f64, and what the
    kernel's rounding is relative to: per row and element the weighted sum of |v| + 8 scales, per row and head the largest
    |scale| * sum |q_d k_td| of the positions it sees."""
    rows, heads, dim = sum(q_lens), q.shape[1], q.shape[2]
    group = heads // k.shape[1]
    out, size, reach = np.zeros((rows, heads, dim)), np.zeros((rows, heads, dim)), np.zeros((rows, heads, 1))
    at = 0
    for b, (n, nq) in enumerate(zip(lens, q_lens)):
        base = sum(lens[:b])
        kb, vb = k[base:base + n].astype(np.float64), v[base:base + n].astype(np.float64)
        pos = np.arange(n - nq, n)
        t = np.arange(n)
        see = t[None] <= pos[:, None]
        if window:
            see &= t[None] > pos[:, None] - window
        some = see.any(1)
        for h in range(heads if n and nq else 0):
            s = np.where(see, q[at:at + nq, h] @ kb[:, h // group].T * scale, -np.inf)
            p = np.zeros_like(s)
            p[some] = np.exp(s[some] - s[some].max(1, keepdims=True))
            p[some] /= p[some].sum(1, keepdims=True)
            out[at:at + nq, h] = p @ vb[:, h // group]
            vh = vb[:, h // group]
            size[at:at + nq, h] = p @ (np.abs(vh) + np.repeat(np.ptp(vh.reshape(n, -1, 64), 2) * 8 / 15, 64, 1))
            reach[at:at + nq, h, 0] = np.where(see, np.abs(q[at:at + nq, h]) @ np.abs(kb[:, h // group]).T * abs(scale), 0).max(1)
        at += nq
    return out, size, reach


def _offsets(dim):
    """Byte and nibble of every (position in block, element) inside a block: K byte, V byte, shift; pair word offsets."""
    t, d = np.meshgrid(np.arange(16), np.arange(dim), indexing="ij")
    g, e = d // 64, d % 64
    u = 2 if dim >= 128 else 1
    kb = (g // u) * (512 * u) + ((t % 2) * 8 + t // 2) * (32 * u) + (e // 16) * (8 * u) + (g % u) * 8 + (e % 16) // 2
    vb = 9 * dim + g * 512 + (e // 8) * 64 + (t // 4) * 16 + (e % 8) // 2 * 4 + t % 4
    return kb, vb, 4 * (d % 2), 8 * dim + g * 64 + t * 4, 17 * dim + g * 64 + t * 4


def decode_position(raw, table, b, p, h, kv_heads, dim, page):
    """One position's key and value of one head, byte by byte."""
    blk = ((int(table[b, p // page]) * kv_heads + h) * (page // 16) + p % page // 16) * 18 * dim
    kb, vb, sh, kp, vp = (o[p % 16] for o in _offsets(dim))
    got = []
    for nib, pair in ((kb, kp), (vb, vp)):
        n = (raw[blk + nib] >> sh) & 15
        s = from_bf16(raw[blk + pair].astype(np.uint16) | raw[blk + pair + 1].astype(np.uint16) << 8)
        z = from_bf16(raw[blk + pair + 2].astype(np.uint16) | raw[blk + pair + 3].astype(np.uint16) << 8)
        got.append(n.astype(F) * s + z)
    return got


def owners(table, lens, num_pages, kv_heads, dim, page):
    """(sequence, position) of every byte of the cache; (-1, -1) where no sequence holds it."""
    own = np.full((num_pages * kv_heads * page // 16 * 18 * dim, 2), -1, np.int64)
    kb, vb, _, kp, vp = _offsets(dim)
    for b, n in enumerate(lens):
        for p in range(n):
            for h in range(kv_heads):
                blk = ((int(table[b, p // page]) * kv_heads + h) * (page // 16) + p % page // 16) * 18 * dim
                for o in (kb, vb, kp, kp + 1, kp + 2, kp + 3, vp, vp + 1, vp + 2, vp + 3):
                    own[blk + o[p % 16]] = (b, p)
    return own
