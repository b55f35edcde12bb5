"""Measured cases of the paged 4-bit KV cache: rotary positions, append with the rotation on the way, attention.

``run`` computes an operator in elementary torch operations (``own`` false) or through the library's entry points
(``own`` true).  The cache is the page format of ``moe_kv4_t`` (include/moe_b200.h): a page holds, per KV head, blocks of
16 positions; a block holds the K nibbles, the K (scale, bias) pairs, the V nibbles and the V pairs.
"""
import math
import random

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
DEV = "cuda"


# ─── cases ──────────────────────────────────────────────────────────────────
def _attn(name, dtype, seqs, q, lens, heads, kv_heads, dim, page, window=0, gate=False, idle=0, mix=1):
    return {"name": name, "op": "attention", "dtype": dtype, "seqs": seqs, "q_min": q[0], "q_max": q[1], "len_min": lens[0],
            "len_max": lens[1], "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "window": window, "gate": gate,
            "idle": idle, "mix": mix}


def _append(name, dtype, seqs, q, lens, kv_heads, dim, rotary, interleaved, page, scaling, mix=1):
    return {"name": name, "op": "append", "dtype": dtype, "seqs": seqs, "q_min": q[0], "q_max": q[1], "len_min": lens[0],
            "len_max": lens[1], "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "interleaved": interleaved, "page": page,
            "scaling": scaling, "idle": 0, "mix": mix}


def _rope(name, dtype, tokens, heads, dim, rotary, interleaved, gap, positions, scaling):
    return {"name": name, "op": "rope", "dtype": dtype, "tokens": tokens, "heads": heads, "dim": dim, "rotary": rotary,
            "interleaved": interleaved, "gap": gap, "positions": positions, "scaling": scaling}


def listed():
    return [
        # one user's decode step early in a conversation, the model's own heads and output gate: latency
        _attn("decode, one short sequence", "f32", 1, (1, 1), (701, 701), 16, 2, 256, 16, gate=True),
        # one user's decode step at a quarter of a million positions: the cache stream
        _attn("decode, one long sequence", "f32", 1, (1, 1), (250001, 250001), 16, 2, 256, 64),
        # a serving batch of sequences of all lengths, two of its slots idle (length 0)
        _attn("decode, ragged batch", "bf16", 48, (1, 1), (100, 16000), 32, 8, 128, 32, idle=2),
        # a speculative loop's verify step: the last token and three drafts of each sequence
        _attn("verify, four tokens each", "bf16", 8, (4, 4), (2000, 9000), 16, 2, 256, 64, gate=True),
        # a long prompt from its first token, the model's own heads
        _attn("prompt, one long", "bf16", 1, (8192, 8192), (8192, 8192), 16, 2, 256, 64, gate=True),
        # short prompts of several users behind a shared prefix, full precision
        _attn("prompts, ragged, f32", "f32", 4, (100, 700), (300, 1500), 16, 2, 256, 16, gate=True),
        # a chunk of a long document under a sliding window, seven query heads to a KV head
        _attn("chunk, window", "bf16", 1, (1001, 1001), (40000, 40000), 14, 2, 64, 16, window=4096),
        # the queries of a decode batch, every head followed by its gate in memory
        _rope("rotate, decode batch", "f32", 48, 16, 256, 64, False, True, 200000, "yarn"),
        # the queries of a long prompt, whole heads in the interleaved layout
        _rope("rotate, long prompt", "bf16", 16384, 32, 128, 128, True, False, 16384, "none"),
        # one new token for every sequence of a decode batch
        _append("append, decode batch", "f32", 48, (1, 1), (100, 16000), 2, 256, 64, False, 32, "yarn"),
        # a prompt's keys and values from its first token, the model's own heads
        _append("append, one prompt", "f32", 1, (8192, 8192), (8192, 8192), 2, 256, 64, False, 64, "none"),
        # chunks of several prompts that begin and end inside pages
        _append("append, ragged chunks", "bf16", 5, (500, 4001), (5000, 30000), 8, 128, 128, True, 16, "linear"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["f32", "bf16"])
    kind = rng.choice(["decode", "decode", "verify", "prompt", "chunk", "rope", "append"])
    dim = rng.choice([64, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 7, 8, 12, 16])
    page = rng.choice([16, 32, 48, 64, 128])
    mix = rng.randrange(1 << 20)
    scaling = rng.choice(["none", "linear", "ntk", "yarn"])
    rotary = rng.choice([dim // 4, dim // 2, dim])
    if kind == "rope":
        c = _rope("", dtype, _log(rng, 1, 16384 * 128 // dim // 2), rng.choice([1, 2, 7, 16, 32]), dim, rotary, rng.random() < 0.5,
                  rng.random() < 0.5, _log(rng, 1000, 200000), scaling)
    elif kind == "append":
        q = _log(rng, 1, 4096)
        c = _append("", dtype, rng.randint(1, 4), (max(1, q // 2), q), (q, 2 * q + 3000), min(kv, 4), dim, rotary, rng.random() < 0.5,
                    page, scaling, mix)
    else:
        window = rng.choice([0, 0, _log(rng, 16, 8192)])
        gate = rng.random() < 0.5
        if kind == "decode":
            seqs = _log(rng, 1, 64)
            top = _log(rng, 1, max(2, min(200000, 48 * 16000 * 8 * 128 // (seqs * kv * dim))))
            c = _attn("", dtype, seqs, (1, 1), (max(1, top // rng.choice([1, 20])), top), kv * group, kv, dim, page, window, gate,
                      rng.choice([0, 1]), mix)
        elif kind == "verify":
            seqs, q = rng.randint(1, 8), rng.randint(2, 9)
            top = _log(rng, 16, 9000)
            c = _attn("", dtype, seqs, (1, q), (16, top), kv * group, kv, dim, page, window, gate, 0, mix)
        elif kind == "prompt":
            q = _log(rng, 17, 1500)
            c = _attn("", dtype, rng.randint(1, 3), (max(1, q // 3), q), (q, q + rng.choice([0, 500])), kv * min(group, 4), kv, dim, page,
                      window, gate, 0, mix)
        else:
            q = rng.randint(100, 600)
            top = _log(rng, 2000, 20000)
            c = _attn("", dtype, 1, (q, q), (top, top), kv * min(group, 4), kv, dim, page, window, gate, 0, mix)
    c.pop("name")
    return c


def _shape(case):
    """Tokens of the call and cached positions (those tokens included) of every sequence; idle ones have 1 and 0."""
    r = random.Random(case["mix"])
    lens, qs = [], []
    for _ in range(case["seqs"]):
        n = _log(r, case["len_min"], case["len_max"])
        lens.append(n)
        qs.append(min(n, r.randint(case["q_min"], case["q_max"])))
    for k in range(case["idle"]):
        at = r.randrange(len(lens) + 1)
        lens.insert(at, 0)
        qs.insert(at, 1)
    return qs, lens


def _pairs(case):
    """(query, position) pairs that the mask leaves, and cached positions that some query sees."""
    pairs = seen = 0
    w = case["window"]
    for q, n in zip(*_shape(case)):
        if n == 0:
            continue
        first = n - q
        if w == 0:
            pairs += q * first + q * (q + 1) // 2
            seen += n
        else:
            p = np.arange(first, n, dtype=np.int64)
            pairs += int(np.minimum(p + 1, w).sum())
            seen += n - max(0, first - w + 1)
    return pairs, seen


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * e + case["tokens"] * (4 + 4 * case["rotary"]), "flops": 3 * n * case["rotary"]}
    qs, _ = _shape(case)
    t = sum(qs)
    per = 18 * case["dim"] // 16  # packed bytes of K and V of one position and head
    if case["op"] == "append":
        n = t * case["kv_heads"]
        return {"bytes": n * (4 * case["dim"] * e + per) + t * 4 * case["rotary"], "flops": n * (3 * case["rotary"] + 8 * case["dim"])}
    pairs, seen = _pairs(case)
    rows = t * case["heads"] * case["dim"] * e
    return {"bytes": seen * case["kv_heads"] * per + rows * (3 if case["gate"] else 2), "flops": 4 * case["dim"] * case["heads"] * pairs}


# ─── the codec and the page format, plain ───────────────────────────────────
def _bf16_bits(x):
    """f32 -> bf16 bit patterns as the packer rounds them: up when bit 15 is set together with bit 0 or bit 16."""
    b = x.contiguous().view(torch.int32)
    up = (b >> 15) & ((b & 0x7FFF) | (b >> 16)) & 1
    return ((b + (up << 16)) >> 16) & 0xFFFF


def _bits_f32(b):
    return (b.to(torch.int32) << 16).view(torch.float32)


def _quantise(x):
    """f32 [..., dim] -> nibbles uint8 [..., dim], scale and bias bits int32 [..., dim / 64]."""
    g = x.reshape(*x.shape[:-1], -1, 64)
    mn, mx = g.amin(-1), g.amax(-1)
    mx = torch.where(mx == mn, mn + 1.0, mx)
    scale = (mx - mn) / torch.full_like(mn, 15.0)  # by a tensor: a division by a number may become a product
    inv = torch.ones_like(scale) / scale
    t = (g - mn[..., None]) * inv[..., None]
    n = torch.trunc(t + 0.5).clamp(0, 15).to(torch.uint8)
    return n.reshape(x.shape), _bf16_bits(scale), _bf16_bits(mn)


def _values(n, s, b):
    g = n.reshape(*n.shape[:-1], -1, 64).float()
    return (g * _bits_f32(s)[..., None] + _bits_f32(b)[..., None]).reshape(n.shape)


def _to_blocks(kq, vq):
    """Quantised K and V [N, 16, dim] (position in block second) -> uint8 [N, 18 * dim]."""
    kn, ks, kb = kq
    vn, vs, vb = vq
    n, _, dim = kn.shape
    groups = dim // 64
    u = min(groups, 2)
    kbyte = (kn[..., 0::2] | (kn[..., 1::2] << 4)).view(n, 8, 2, groups // u, u, 4, 8)  # block, t / 2, t % 2, pair, u, c, byte
    kbyte = kbyte.permute(0, 3, 2, 1, 5, 4, 6).reshape(n, -1)
    vbyte = (vn[..., 0::2] | (vn[..., 1::2] << 4)).view(n, 4, 4, groups, 8, 4)           # block, quad, t % 4, group, row, x
    vbyte = vbyte.permute(0, 3, 4, 1, 5, 2).reshape(n, -1)

    def pairs(s, b):
        w = torch.stack([s & 255, s >> 8, b & 255, b >> 8], -1).to(torch.uint8)          # block, t, group, 4
        return w.permute(0, 2, 1, 3).reshape(n, -1)

    return torch.cat([kbyte, pairs(ks, kb), vbyte, pairs(vs, vb)], 1)


def _from_blocks(blk, dim):
    """uint8 [N, 18 * dim] -> K and V values, f32 [N, 16, dim]."""
    n, groups = blk.shape[0], dim // 64
    u = min(groups, 2)
    kw, kp, vw, vp = blk.split([8 * dim, dim, 8 * dim, dim], 1)
    kbyte = kw.reshape(n, groups // u, 2, 8, 4, u, 8).permute(0, 3, 2, 1, 5, 4, 6).reshape(n, 16, dim // 2)
    vbyte = vw.reshape(n, groups, 8, 4, 4, 4).permute(0, 3, 5, 1, 2, 4).reshape(n, 16, dim // 2)

    def values(byte, pair):
        nib = torch.stack([byte & 15, byte >> 4], -1).reshape(n, 16, dim)
        w = pair.reshape(n, groups, 16, 4).permute(0, 2, 1, 3).to(torch.int32)
        return _values(nib, w[..., 0] | (w[..., 1] << 8), w[..., 2] | (w[..., 3] << 8))

    return values(kbyte, kp), values(vbyte, vp)


def _table(n_positions, rotary, scaling):
    """cos then sin of every position's angles, f32 [n_positions, rotary]; angles in 64 bits."""
    theta, factor, original = 1.0e7, 4.0, 8192
    i = torch.arange(rotary // 2, dtype=torch.float64, device=DEV)
    if scaling == "ntk":
        theta = theta * factor ** (rotary / (rotary - 2))
    freq = theta ** (-2.0 * i / rotary)
    mul = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        turn = lambda n: rotary * math.log(original / (n * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(turn(32.0)), 0), min(math.ceil(turn(1.0)), rotary - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq / factor * ramp + freq * (1 - ramp)
        mul = 0.1 * math.log(factor) + 1.0
    a = torch.arange(n_positions, dtype=torch.float64, device=DEV)[:, None] * freq
    return torch.cat([a.cos() * mul, a.sin() * mul], 1).float()


# ─── inputs ─────────────────────────────────────────────────────────────────
def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    dt = DT[case["dtype"]]
    st = {"case": case}
    if case["op"] == "rope":
        t, h, d = case["tokens"], case["heads"], case["dim"]
        # with a gap every head is followed by as many elements of something else (its output gate)
        st["x"] = normal(t, h, 2 * d if case["gap"] else d).to(dt)
        st["pos"] = torch.randint(0, case["positions"], (t,), generator=g, device=DEV, dtype=torch.int32)
        st["table"] = _table(case["positions"], case["rotary"], case["scaling"])
        return st
    qs, lens = _shape(case)
    kv, d, page = case["kv_heads"], case["dim"], case["page"]
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    st["table"], st["n_pages"] = table, n_pages
    st["q_start"] = torch.tensor(np.concatenate([[0], np.cumsum(qs)]), dtype=torch.int32, device=DEV)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    st["seq"] = torch.tensor(np.repeat(np.arange(len(qs)), qs), dtype=torch.int64, device=DEV)
    st["tokens"], st["longest"], st["longest_q"] = sum(qs), max(lens), max(qs)
    tokens = st["tokens"]
    # keys: a spread of channel sizes; values: near normal
    spread = torch.exp(0.4 * normal(kv, 1, d))
    if case["op"] == "append":
        st["pages"] = torch.zeros(n_pages, kv, page // 16, 18 * d, dtype=torch.uint8, device=DEV)
        st["k"] = (normal(tokens, kv, d) * spread.reshape(1, kv, d)).to(dt)
        st["v"] = normal(tokens, kv, d).to(dt)
        st["rope"] = _table(max(lens), case["rotary"], case["scaling"])
        return st
    pages = torch.empty(n_pages, kv, page // 16, 18 * d, dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 26) // (kv * page * d))
    for a in range(0, n_pages, step):
        n = min(step, n_pages - a)
        k = normal(n, kv, page, d) * spread
        v = normal(n, kv, page, d)
        pages[a:a + n] = _to_blocks(_quantise(k.reshape(-1, 16, d)), _quantise(v.reshape(-1, 16, d))).view(n, kv, page // 16, 18 * d)
    st["pages"] = pages
    st["q"] = (1.5 * normal(tokens, case["heads"], d)).to(dt)
    st["gate"] = normal(tokens, case["heads"], d).to(dt) if case["gate"] else None
    return st


# ─── the framework's calls ──────────────────────────────────────────────────
_engine = _stream = _made = _done = None


def _eng():
    global _engine, _stream, _made, _done
    if _engine is None:
        from moe_infer_b200.native import Dims, NativeEngine
        _engine = NativeEngine(Dims(num_experts=4, top_k=4, num_layers=1))
        _stream = torch.cuda.ExternalStream(_engine.stream())
        _made, _done = torch.cuda.Event(), torch.cuda.Event()
    return _engine


def _run_own(st):
    """The engine has a stream of its own: it waits for what torch's stream has made of the inputs (and for earlier users of the
    outputs' memory), and torch's stream waits for the results."""
    eng, mine = _eng(), torch.cuda.current_stream()
    _made.record(mine)
    _stream.wait_event(_made)
    out = _calls(st, eng)
    _done.record(_stream)
    mine.wait_event(_done)
    return out


def _calls(st, eng):
    from moe_infer_b200.native import Kv4Batch, Kv4Cache, RopeTable
    case = st["case"]
    dtype = 0 if case["dtype"] == "f32" else 1  # MOE_DT_F32, MOE_DT_BF16
    if case["op"] == "rope":
        x, d = st["x"], case["dim"]
        out = torch.empty(case["tokens"], case["heads"], d, dtype=x.dtype, device=DEV)
        rope = RopeTable(st["table"].data_ptr(), case["positions"], case["rotary"], case["interleaved"])
        eng.rope_dev(rope, x.data_ptr(), out.data_ptr(), st["pos"].data_ptr(), dtype, case["tokens"], case["heads"], d,
                     x_strides=(x.stride(0), x.stride(1)))
        return out
    kv, d = case["kv_heads"], case["dim"]
    cache = Kv4Cache(st["pages"].data_ptr(), st["n_pages"], case["page"], kv, d)
    batch = Kv4Batch(st["q_start"].data_ptr(), st["lens"].data_ptr(), st["table"].data_ptr(), st["lens"].shape[0], st["tokens"],
                     st["table"].shape[1], st["longest"], st["longest_q"])
    if case["op"] == "append":
        k, v = st["k"], st["v"]
        rope = RopeTable(st["rope"].data_ptr(), st["rope"].shape[0], case["rotary"], case["interleaved"])
        eng.kv4_append_dev(cache, batch, k.data_ptr(), v.data_ptr(), dtype, rope=rope)
        ko, vo = torch.empty_like(k), torch.empty_like(v)
        eng.kv4_gather_dev(cache, batch, ko.data_ptr(), vo.data_ptr(), dtype)
        return {"k": ko, "v": vo}
    q, gate = st["q"], st["gate"]
    out = torch.empty_like(q)
    eng.kv4_attention_dev(cache, batch, q.data_ptr(), out.data_ptr(), dtype, case["heads"], scale=1.0 / math.sqrt(d), window=case["window"],
                          gate=gate.data_ptr() if gate is not None else 0)
    return out


# ─── the plain form ─────────────────────────────────────────────────────────
def _rotate(x, cs, interleaved):
    """x f32 [T, H, dim], cs f32 [T, rotary]."""
    r = cs.shape[1]
    c, s = cs[:, None, :r // 2], cs[:, None, r // 2:]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    na, nb = a * c - b * s, a * s + b * c
    turned = torch.stack([na, nb], -1).flatten(-2) if interleaved else torch.cat([na, nb], -1)
    return torch.cat([turned, x[..., r:]], -1)


def run(st):
    if own:
        return _run_own(st)
    case = st["case"]
    dt = DT[case["dtype"]]
    if case["op"] == "rope":
        x = st["x"][..., :case["dim"]].float()
        return _rotate(x, st["table"][st["pos"].long()], case["interleaved"]).to(dt)
    kv, d, page = case["kv_heads"], case["dim"], case["page"]
    seq, lens, q_start = st["seq"], st["lens"].long(), st["q_start"].long()
    tokens = st["tokens"]
    j = torch.arange(tokens, device=DEV) - q_start[seq]
    n_q = q_start[1:] - q_start[:-1]
    pos = lens[seq] - n_q[seq] + j
    if case["op"] == "append":
        k = _rotate(st["k"].float(), st["rope"][pos], case["interleaved"])
        return {"k": _values(*_quantise(k)).to(dt), "v": _values(*_quantise(st["v"].float())).to(dt)}
    blocks = st["pages"][st["table"].clamp(min=0).long()]                    # [B, pages, kv, page / 16, bytes]
    n_seq, per = blocks.shape[0], blocks.shape[1] * page
    k, v = _from_blocks(blocks.reshape(-1, 18 * d), d)
    kv_order = lambda x: x.view(n_seq, -1, kv, page, d).transpose(1, 2).reshape(n_seq, kv, per, d)  # noqa: E731
    k, v = kv_order(k), kv_order(v)
    heads, group, q_max = case["heads"], case["heads"] // kv, st["longest_q"]
    q = torch.zeros(n_seq, q_max, heads, d, device=DEV)
    q[seq, j] = st["q"].float()
    q = q.view(n_seq, q_max, kv, group, d).permute(0, 2, 3, 1, 4).reshape(n_seq, kv, group * q_max, d)
    s = torch.matmul(q, k.transpose(2, 3)).view(n_seq, kv, group, q_max, per) * (1.0 / math.sqrt(d))
    at = (lens - n_q)[:, None] + torch.arange(q_max, device=DEV)            # [B, q]
    t = torch.arange(per, device=DEV)
    see = t <= at[..., None]
    if case["window"]:
        see &= t > at[..., None] - case["window"]
    s = s.masked_fill(~see[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n_seq, kv, group * q_max, per), v).view(n_seq, kv, group, q_max, d)
    o = o / torch.where(total == 0, torch.ones_like(total), total)
    o = o.permute(0, 3, 1, 2, 4).reshape(n_seq, q_max, heads, d)[seq, j]
    if st["gate"] is not None:
        o = o / (1.0 + torch.exp(-st["gate"].float()))
    return o.to(dt)


# ─── the definition in 64 bits ──────────────────────────────────────────────
def _exact_angles(pos, rotary, scaling):
    theta, factor, original = 1.0e7, 4.0, 8192.0
    mul, freq = 1.0, []
    if scaling == "ntk":
        theta *= factor ** (rotary / (rotary - 2.0))
    if scaling == "yarn":
        edge = [rotary * math.log(original / (n * 2.0 * math.pi)) / (2.0 * math.log(theta)) for n in (32.0, 1.0)]
        low, high = max(0, math.floor(edge[0])), min(rotary - 1, math.ceil(edge[1]))
        mul = 1.0 + 0.1 * math.log(factor)
    for i in range(rotary // 2):
        f = math.pow(theta, -2.0 * i / rotary)
        if scaling == "linear":
            f /= factor
        if scaling == "yarn":
            w = min(1.0, max(0.0, (i - low) / max(high - low, 1e-3)))
            f = f * (1.0 - w) + f * w / factor
        freq.append(f)
    a = np.asarray(pos, np.float64)[:, None] * np.array(freq)[None]
    return np.cos(a) * mul, np.sin(a) * mul


def _exact_turn(x, c, s, interleaved):
    """numpy [T, H, dim], in the type of its arguments, every operation rounded on its own."""
    r = 2 * c.shape[1]
    y = x.copy()
    ia = np.arange(0, r, 2) if interleaved else np.arange(r // 2)
    ib = ia + (1 if interleaved else r // 2)
    a, b, c, s = x[..., ia], x[..., ib], c[:, None], s[:, None]
    y[..., ia] = a * c - b * s
    y[..., ib] = a * s + b * c
    return y


def _exact_codec(x):
    """The value that every element of f32 [..., dim] is held as: the codec is defined in f32 steps."""
    f = np.float32
    x = x.reshape(-1, 64)
    lo, hi = x.min(1), x.max(1)
    hi = np.where(hi == lo, lo + f(1), hi)
    step = ((hi - lo) / f(15)).astype(f)
    t = ((x - lo[:, None]) * (f(1) / step)[:, None]).astype(f) + f(0.5)
    n = np.clip(np.floor(np.maximum(t, f(0))), 0, 15)

    def rounded(v):
        u = v.astype(f).view(np.uint32)
        up = ((u >> 15) & 1) & ((u & 1) | ((u >> 16) & 1))
        return (((u + (up << 16)) >> 16) << 16).astype(np.uint32).view(f).astype(np.float64)

    return n * rounded(step)[:, None] + rounded(lo)[:, None]


def _exact_rows(st, b, h, n):
    """K and V of one sequence and head as f64 [n, dim], byte by byte from the page format."""
    case = st["case"]
    d, page = case["dim"], case["page"]
    t = torch.arange(n, device=DEV)
    at = st["table"][b].long()[t // page] * case["kv_heads"] + h
    base = (at * (page // 16) + t % page // 16) * (18 * d)
    tb = (t % 16)[:, None]
    raw = st["pages"].view(-1)
    e = torch.arange(d, device=DEV)[None]
    g, in_g = e // 64, e % 64
    u = 2 if d >= 128 else 1
    k_at = (g // u) * (512 * u) + (tb % 2 * 8 + tb // 2) * (32 * u) + in_g // 16 * (8 * u) + g % u * 8 + in_g % 16 // 2
    v_at = g * 512 + in_g // 8 * 64 + tb // 4 * 16 + in_g % 8 // 2 * 4 + tb % 4
    got = []
    for where, sb in ((k_at, 8 * d), (9 * d + v_at, 17 * d)):
        nib = (raw[base[:, None] + where].long() >> (4 * (e % 2))) & 15
        w = base[:, None] + sb + torch.arange(d // 64, device=DEV)[None] * 64 + tb * 4
        half = lambda o: ((raw[w + o].to(torch.int32) | (raw[w + o + 1].to(torch.int32) << 8)) << 16).view(torch.float32).double()  # noqa: E731
        got.append(nib.double() * half(0).repeat_interleave(64, 1) + half(2).repeat_interleave(64, 1))
    return got


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        c, s = _exact_angles(st["pos"].cpu().numpy(), case["rotary"], case["scaling"])
        x = st["x"][..., :case["dim"]].double().cpu().numpy()
        return torch.from_numpy(_exact_turn(x, c, s, case["interleaved"]))
    qs, lens = _shape(case)
    if case["op"] == "append":
        pos = np.concatenate([np.arange(n - q, n) for q, n in zip(qs, lens)])
        r = case["rotary"]
        cs = st["rope"].cpu().numpy()[pos]  # the table is an input; the rotation and the codec are f32 steps by definition
        k = _exact_turn(st["k"].float().cpu().numpy(), cs[:, :r // 2], cs[:, r // 2:], case["interleaved"])
        v = st["v"].float().cpu().numpy()
        return {"k": torch.from_numpy(_exact_codec(k).reshape(k.shape)), "v": torch.from_numpy(_exact_codec(v).reshape(v.shape))}
    heads, kv, d = case["heads"], case["kv_heads"], case["dim"]
    group = heads // kv
    out = torch.zeros(st["tokens"], heads, d, dtype=torch.float64, device=DEV)
    row = 0
    for b, (nq, n) in enumerate(zip(qs, lens)):
        for h in range(kv if n else 0):
            k, v = _exact_rows(st, b, h, n)
            p = torch.arange(n - nq, n, device=DEV)[:, None]
            t = torch.arange(n, device=DEV)[None]
            hidden = (t > p) | ((t <= p - case["window"]) if case["window"] else False)
            for x in range(h * group, (h + 1) * group):
                s = st["q"][row:row + nq, x].double() @ k.T / math.sqrt(d)
                out[row:row + nq, x] = torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ v
        row += nq
    if st["gate"] is not None:
        out = out * torch.sigmoid(st["gate"].double())
    return out
