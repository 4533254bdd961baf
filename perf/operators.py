"""What the operators of long-context serving are measured on: a cache of keys and values held in 4 bits, and attention
that sees a window of recent tokens and a few first ones.

Three operators, each a call that an attention layer makes once per step:

* ``store``: queries and keys of a step are rotated by their positions, the queries handed on, keys and values rounded to
  4 bits (a whole number from -7 to 7 and, for every 32 values of a head, one scale: a bfloat16 of 5 significant bits, so that
  the products are bfloat16 numbers too) and written to their places in the cache's pages; what they then hold is read back.
* ``attend4``: causal attention of the step's queries over such a cache: single tokens of many requests, or portions of
  prompts, over all keys, or over a window and the first tokens.
* ``attend``: attention over a window and the first tokens of an ordinary cache, in the compute type.

The layout of a 4-bit page is the cache's own: for a kv head and 16 tokens, 16 rows of keys' codes, 16 of values', 16 rows
of the keys' scales, 16 of the values'.  A code is the number plus 8.  Of a key's 32 * G dims, dim 32 g + 8 t + i is nibble
i of 32-bit word t * G + g of its row; of a value's, dim 16 i + 2 e + j is nibble j of byte e * 2 G + i.

Head layouts and lengths are those of the configurations the engine is specified on (the small one of the tests, Llama 3.2
1B, Llama 3.1 8B) and a few others that a head count and size can take.  Pages hold 16 tokens and lie in no order.
"""
from __future__ import annotations

import math
import types

import numpy as np
import torch

own = False

DEV = "cuda:0"
PAGE = 16
GROUP = 32                       # dims of a head that share a scale
THETA = 500000.0

# query heads, kv heads, head size
HEADS = {"small": (4, 1, 32), "1b": (32, 8, 64), "8b": (32, 8, 128), "even": (12, 12, 96), "shared": (16, 1, 128),
         "wide": (8, 4, 256)}


def listed():
    return [
        # A step of four tokens of the small model, in 32-bit: nothing but latency.
        dict(name="store_small", kind="store", heads="small", dtype="float32", requests=4, shortest=3, longest=70, tokens=1),
        # A decode step of 64 requests at 1B sizes: their new keys and values.
        dict(name="store_decode_1b", kind="store", heads="1b", dtype="bfloat16", requests=64, shortest=100, longest=4000, tokens=1),
        # A prompt portion of an odd length, late in a long prompt, at 8B sizes.
        dict(name="store_prompt_8b", kind="store", heads="8b", dtype="bfloat16", requests=1, shortest=30000, longest=30000,
             tokens=2011),
        # The smallest call: one request at the start of its answer.
        dict(name="single_short", kind="attend4", heads="1b", dtype="bfloat16", requests=1, shortest=37, longest=37, tokens=1,
             window=0, first=0),
        # The engine's headline with the cache in 4 bits: 8 requests at 4,096 tokens, 1B sizes.
        dict(name="decode_1b_8", kind="attend4", heads="1b", dtype="bfloat16", requests=8, shortest=4096, longest=4096, tokens=1,
             window=0, first=0),
        # Serving under load at 8B sizes: 64 requests of ragged lengths.
        dict(name="decode_8b_64", kind="attend4", heads="8b", dtype="bfloat16", requests=64, shortest=1000, longest=8100, tokens=1,
             window=0, first=0),
        # One conversation at the longest context the configurations allow.
        dict(name="decode_long", kind="attend4", heads="8b", dtype="bfloat16", requests=1, shortest=131072, longest=131072, tokens=1,
             window=0, first=0),
        # Endless conversations: 32 requests far along, each with its last 2,000 tokens and its first 4; 32-bit rows.
        dict(name="window_32bit", kind="attend4", heads="1b", dtype="float32", requests=32, shortest=2500, longest=60000, tokens=1,
             window=2000, first=4),
        # A short question behind a long document.
        dict(name="question", kind="attend4", heads="8b", dtype="bfloat16", requests=1, shortest=30040, longest=30040, tokens=40,
             window=0, first=0),
        # A later portion of a long prompt, an odd number of tokens.
        dict(name="portion_8b", kind="attend4", heads="8b", dtype="bfloat16", requests=1, shortest=6107, longest=6107, tokens=2011,
             window=0, first=0),
        # An ordinary cache, decoded far beyond its window: 64 requests at 8B sizes.
        dict(name="first_decode", kind="attend", heads="8b", dtype="bfloat16", requests=64, shortest=500, longest=20000, tokens=1,
             window=1024, first=4),
        # ... and a prompt portion there.
        dict(name="first_portion", kind="attend", heads="1b", dtype="bfloat16", requests=1, shortest=8000, longest=8000, tokens=2000,
             window=1024, first=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "attend4", "attend4", "attend4", "attend"])
    c = dict(kind=kind, heads=rng.choice(["small", "1b", "1b", "8b", "8b", "even", "shared", "wide"]),
             dtype=rng.choice(["bfloat16"] * 4 + ["float32"]))
    prompt = rng.random() < 0.4
    c["requests"] = rng.randint(1, 3) if prompt else _log(rng, 1, 64)
    c["tokens"] = _log(rng, 2, 1200 // c["requests"]) if prompt else 1
    budget = 130000 if kind == "attend4" and not prompt else 15000
    c["longest"] = c["tokens"] + _log(rng, 3, max(4, budget // c["requests"]))
    c["shortest"] = rng.randint(c["tokens"], c["longest"])
    if kind != "store":
        windowed = kind == "attend" or rng.random() < 0.4
        c["window"] = _log(rng, 1, 2500) if windowed else 0
        c["first"] = rng.choice([1, 4, 5, 16, 64, 100]) if windowed else 0
    return c


# ------------------------------------------------------------------ inputs
def _dtype(case):
    return torch.float32 if case["dtype"] == "float32" else torch.bfloat16


def _lengths(case):
    """The requests' lengths after the step, spread evenly and in no order."""
    n, lo, hi = case["requests"], case["shortest"], case["longest"]
    return [hi] if n == 1 else [lo + (hi - lo) * ((7 * i + 3) % n) // (n - 1) for i in range(n)]


def _held(case):
    """Per request the pages of positions that the step can see or writes: (first page numbers, then those of the window)."""
    W, F, n = case.get("window", 0), case.get("first", 0), case["tokens"]
    held = []
    for L in _lengths(case):
        if case["kind"] == "store":
            held.append(list(range((L - n) // PAGE, -(-L // PAGE))))
            continue
        lo = max(0, L - n - W + 1) if W else 0
        near = list(range(lo // PAGE, -(-L // PAGE)))
        held.append([p for p in range(-(-min(F, L) // PAGE)) if p < lo // PAGE] + near)
    return held


def _scale(largest):
    """A seventh of a group's largest value, in 32-bit, rounded to 5 significant bits."""
    bits = (largest.double() / 7).float().view(torch.int32)
    return ((bits + 0x3ffff + (bits >> 19 & 1)) & ~0x7ffff).view(torch.float32)


def _quantised(x):
    """Codes (0 to 15) and bfloat16 scales of x [..., dims], groups of 32 dims."""
    g = x.unflatten(-1, (-1, GROUP))
    s = _scale(g.abs().amax(-1, keepdim=True))
    n = torch.round(g / s)
    return (n.clamp(-7, 7) + 8).to(torch.uint8).flatten(-2), s.squeeze(-1).bfloat16()


def _packed(kc, ks, vc, vs):
    """Pages [pages, kv heads, page / 16, bytes] from codes [pages, kv heads, page, dims] and scales [..., dims / 32]."""
    P, H, S, D = kc.shape
    G = D // GROUP
    k = kc.view(P, H, S, G, 4, 4, 2)
    k = (k[..., 0] | k[..., 1] << 4).transpose(3, 4).reshape(P, H, S // 16, 16 * D // 2)
    v = vc.view(P, H, S, 2 * G, 8, 2)
    v = (v[..., 0] | v[..., 1] << 4).transpose(3, 4).reshape(P, H, S // 16, 16 * D // 2)
    s = [t.contiguous().view(P, H, S // 16, 16 * G).view(torch.uint8) for t in (ks, vs)]
    return torch.cat([k, v] + s, dim=-1).contiguous()


def _drawn(shape, g, spread):
    """Values as projections give them: each channel with a size of its own."""
    size = torch.exp(spread * torch.randn(shape[-1], device=DEV, generator=g))
    return torch.randn(shape, device=DEV, generator=g) * size


def prepare(case, seed):
    nh, nkv, hd = HEADS[case["heads"]]
    dt = _dtype(case)
    g = torch.Generator(device=DEV).manual_seed(1000003 * (seed + 1))
    lens, held = _lengths(case), _held(case)
    R, n = case["requests"], case["tokens"]
    T = R * n
    q_len, kv_len = np.full(R, n, dtype=np.int32), np.array(lens, dtype=np.int32)
    start = (np.arange(R + 1) * n).astype(np.int32)
    positions = np.concatenate([np.arange(L - n, L) for L in lens]).astype(np.int32)

    def dev(a):
        return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)

    # the step as the engine describes it to its kernels
    ctx = types.SimpleNamespace(
        n_tokens=T, n_requests=R, max_q_len=n, max_kv_len=int(kv_len.max()), h_q_len=q_len, h_kv_len=kv_len, h_q_start=start,
        h_table_rows=np.arange(R, dtype=np.int32), positions=dev(positions), token_req=dev(np.repeat(np.arange(R, dtype=np.int32), n)),
        q_start=dev(start), kv_len=dev(kv_len), table_rows=dev(np.arange(R, dtype=np.int32)))
    P = sum(map(len, held))
    ids = torch.randperm(P, generator=torch.Generator().manual_seed(seed)).to(torch.int32).numpy()
    table = np.full((R, -(-max(lens) // PAGE)), -1, dtype=np.int32)
    at = 0
    for r, pages in enumerate(held):
        table[r, pages] = ids[at:at + len(pages)]
        at += len(pages)
    state = dict(case=case, ctx=ctx, table=dev(table), scale=1.0 / math.sqrt(hd),
                 qkv=_drawn((T, nh + 2 * nkv, hd), g, 0.4).flatten(1).to(dt))
    if case["kind"] == "attend":
        state["pages"] = tuple(_drawn((P, nkv, PAGE, hd), g, 0.3).to(dt) for _ in range(2))
    else:
        state["pages"] = _packed(*_quantised(_drawn((P, nkv, PAGE, hd), g, 0.3)), *_quantised(_drawn((P, nkv, PAGE, hd), g, 0.1)))
    if case["kind"] == "store":
        state["inv_freq"] = torch.pow(torch.tensor(THETA, dtype=torch.float64), -torch.arange(0, hd, 2, dtype=torch.float64) / hd).float().to(DEV)
        state["q"] = torch.empty(T, nh * hd, dtype=dt, device=DEV)
        state["rows"] = ctx.token_req                      # the block-table row of each token
        state["k"], state["v"] = (torch.empty(T, nkv, hd, dtype=dt, device=DEV) for _ in range(2))
    else:
        state["out"] = torch.empty(T, nh * hd, dtype=dt, device=DEV)
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    nh, nkv, hd = HEADS[case["heads"]]
    if own:
        return _run_own(state, case, nh, nkv, hd)
    if case["kind"] == "store":
        return _plain_store(state, nh, nkv, hd)
    return _plain_attention(state, case, nh, nkv, hd)


def _run_own(state, case, nh, nkv, hd):
    from llm_singularity_b200 import kernels as ops
    from llm_singularity_b200.parts.base import KV4CacheView, KVCacheView
    ctx, qkv = state["ctx"], state["qkv"]
    if case["kind"] == "attend":
        cache = KVCacheView(state["pages"][0], state["pages"][1], state["table"], PAGE, case["window"], 0)
        ops.paged_attention(qkv, nh, nkv, hd, ctx, cache, state["scale"], case["window"], state["out"], first=case["first"])
        return state["out"]
    cache = KV4CacheView(state["pages"], state["table"], PAGE, case.get("window") or None, 0)
    if case["kind"] == "attend4":
        ops.paged_attention_kv4(qkv, nh, nkv, hd, ctx, cache, state["scale"], case["window"], state["out"], first=case["first"])
        return state["out"]
    ops.rope_kv4_store(qkv, nh, nkv, hd, ctx, cache, state["inv_freq"], hd, state["q"])
    ops.read_kv4(cache, nkv, hd, state["rows"], ctx.positions, state["k"], state["v"])
    return dict(q=state["q"], k=state["k"], v=state["v"])


def _plain_rounded(x, dtype):
    """The values that x [..., dims] stands for in 4 bits; next to a border between two codes 32 bits would not do."""
    g = x.unflatten(-1, (-1, GROUP)).double()
    s = _scale(g.abs().amax(-1, keepdim=True)).double()
    n = torch.where(s > 0, torch.round(g / s).clamp(-7, 7), torch.zeros_like(g))
    return (n * s).flatten(-2).to(dtype)


def _plain_store(state, nh, nkv, hd):
    qkv, ctx = state["qkv"], state["ctx"]
    x = qkv.view(-1, nh + 2 * nkv, hd)
    angle = ctx.positions.double()[:, None] * state["inv_freq"].double()
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = x[:, :nh + nkv].double().chunk(2, -1)
    turned = torch.cat([a * c - b * s, a * s + b * c], -1).float().to(qkv.dtype)
    return dict(q=turned[:, :nh].flatten(1), k=_plain_rounded(turned[:, nh:], qkv.dtype), v=_plain_rounded(x[:, nh + nkv:], qkv.dtype))


def _plain_pages(pages, hd):
    """Keys and values [pages, kv heads, page, dims] in 32-bit of 4-bit pages."""
    P, H, S, _ = pages.shape
    G, half = hd // GROUP, 8 * hd
    k = pages[..., :half].reshape(P, H, S * 16, 4, G, 4).transpose(3, 4)
    v = pages[..., half:2 * half].reshape(P, H, S * 16, 8, 2 * G).transpose(3, 4)
    s = pages[..., 2 * half:].contiguous().view(torch.bfloat16).float().view(P, H, S, 2, 16, G).transpose(2, 3)
    s = s.reshape(P, H, 2, S * 16, G, 1).unbind(2)
    k, v = (torch.stack([t & 15, t >> 4], -1).reshape(P, H, S * 16, G, GROUP).float() - 8.0 for t in (k, v))
    return (k * s[0]).flatten(-2), (v * s[1]).flatten(-2)


def _plain_attention(state, case, nh, nkv, hd):
    ctx, qkv, W, F = state["ctx"], state["qkv"], case["window"], case["first"]
    R, n = ctx.n_requests, case["tokens"]
    K, V = _plain_pages(state["pages"], hd) if case["kind"] == "attend4" else (p.float() for p in state["pages"])
    # the positions that a request's rows can see: the first tokens, and from the oldest row's window on
    L = ctx.kv_len.long()[:, None]
    lo = (L - n - W + 1).clamp_min(0) if W else torch.zeros_like(L)
    few = lo.clamp_max(F)
    most = case["longest"] if not W else min(case["longest"], F + W + n - 1)
    i = torch.arange(most, device=qkv.device)[None]
    pos = torch.where(i < few, i, i - few + lo)
    there = pos < L
    pos = torch.minimum(pos, L - 1)
    page, off = state["table"].gather(1, pos // PAGE).long(), pos % PAGE
    K, V = (t[page, :, off].permute(0, 2, 1, 3) for t in (K, V))          # [requests, kv heads, positions, dims]
    q = qkv[:, :nh * hd].float().view(R, n, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4)
    s = torch.matmul(q.flatten(2, 3), K.transpose(2, 3)).view(R, nkv, nh // nkv, n, most) * state["scale"]
    own_pos = (L - n + torch.arange(n, device=qkv.device))[:, :, None]
    sees = there[:, None] & (pos[:, None] <= own_pos)
    if W:
        sees = sees & ((pos[:, None] > own_pos - W) | (pos[:, None] < F))
    s = s.masked_fill(~sees[:, None, None], -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul((e / e.sum(-1, keepdim=True)).flatten(2, 3), V).view(R, nkv, nh // nkv, n, hd)
    return o.permute(0, 3, 1, 2, 4).reshape(R * n, nh * hd).to(qkv.dtype)


# ------------------------------------------------------------------ what a pass cannot do without
def _seen(case):
    """(positions that a request's rows see together, pairs of a row and a position that it sees), over all requests."""
    W, F, n = case["window"], case["first"], case["tokens"]
    together = pairs = 0
    for L in _lengths(case):
        lo = max(0, L - n - W + 1) if W else 0
        together += min(F, lo) + L - lo
        p = np.arange(L - n, L)
        near = np.maximum(0, p - W + 1) if W else np.zeros_like(p)
        pairs += int((p - near + 1 + np.minimum(F, near)).sum())
    return together, pairs


def work(case):
    nh, nkv, hd = HEADS[case["heads"]]
    e = 4 if case["dtype"] == "float32" else 2
    T = case["requests"] * case["tokens"]
    if case["kind"] == "store":
        # projections in, queries out, codes and scales out; then what they stand for
        four_bits = T * 2 * nkv * (hd // 2 + hd // 16)
        return {"bytes": T * (nh + 2 * nkv) * hd * e + T * nh * hd * e + four_bits + T * 2 * nkv * hd * e,
                "flops": T * (6 * (nh + nkv) * hd + 8 * nkv * hd)}
    together, pairs = _seen(case)
    row = 2 * (hd // 2 + hd // 16) if case["kind"] == "attend4" else 2 * hd * e
    return {"bytes": together * nkv * row + 2 * T * nh * hd * e, "flops": 4 * pairs * nh * hd}


# ------------------------------------------------------------------ from the definition, in 64 bits
def _exact_row(codes, scales, order):
    """One head's vector for each token: codes [tokens, dims] as stored bytes, `order`: (byte, shift) of each dim."""
    byte, shift = order
    n = torch.div(codes.long()[:, byte], 2 ** shift, rounding_mode="floor") % 16 - 8
    return n.double() * scales.double().repeat_interleave(GROUP, 1)


def _exact_orders(hd):
    G = hd // GROUP
    d = torch.arange(hd, device=DEV)
    word = (d % 32 // 8) * G + d // 32
    return (4 * word + d % 8 // 2, 4 * (d % 2)), (d % 16 // 2 * 2 * G + d // 16, 4 * (d % 2))


def exact(case, seed):
    nh, nkv, hd = HEADS[case["heads"]]
    state = prepare(case, seed)
    dt, n = _dtype(case), case["tokens"]
    x = state["qkv"].double().view(-1, nh + 2 * nkv, hd)
    if case["kind"] == "store":
        half = hd // 2
        turn = torch.polar(torch.ones(1, dtype=torch.float64, device=DEV),
                           state["ctx"].positions.double()[:, None] * state["inv_freq"].double()[None])[:, None]
        z = torch.complex(x[:, :nh + nkv, :half].contiguous(), x[:, :nh + nkv, half:].contiguous()) * turn
        qk = torch.cat([z.real, z.imag], -1)

        def held(y):
            """What 4 bits hold of y, a scale for every 32 dims: 15 values from -7 to 7 times the scale."""
            y = y.float().to(dt).double().reshape(y.shape[0], nkv, -1, GROUP)
            part, power = np.frexp(np.float32(y.abs().max(-1).values.cpu().numpy() / 7.0).astype(np.float64))
            scale = torch.from_numpy(np.ldexp(np.rint(part * 32), power - 5)).to(y.device)[..., None]
            scale = torch.where(scale > 0, scale, 1.0)
            return (torch.round(y / scale).clamp(-7, 7) * scale).reshape(y.shape[0], nkv, hd)

        return dict(q=qk[:, :nh].reshape(-1, nh * hd), k=held(qk[:, nh:]), v=held(x[:, nh + nkv:]))
    out = torch.empty(x.shape[0], nh, hd, dtype=torch.float64, device=DEV)
    table, orders = state["table"].cpu().numpy(), _exact_orders(hd)
    W, F, group, G = case["window"], case["first"], nh // nkv, hd // GROUP
    for r, L in enumerate(_lengths(case)):
        lo = max(0, L - n - W + 1) if W else 0
        seen = np.concatenate([np.arange(min(F, lo)), np.arange(lo, L)])
        page, off = (torch.from_numpy(a).to(DEV).long() for a in (table[r, seen // PAGE], seen % PAGE))
        pos = torch.from_numpy(seen).to(DEV)
        own_pos = torch.arange(L - n, L, device=DEV)
        hidden = pos[None] > own_pos[:, None]
        if W:
            hidden |= (pos[None] <= own_pos[:, None] - W) & (pos[None] >= F)
        for h in range(nkv):
            if case["kind"] == "attend":
                k, v = (p[page, h, off].double() for p in state["pages"])
            else:
                raw, row = state["pages"][page, h, 0], hd // 2
                part = [raw[:, a:a + 16 * w].view(-1, 16, w)[torch.arange(len(page)), off].contiguous()
                        for a, w in ((0, row), (16 * row, row), (32 * row, 2 * G), (32 * row + 32 * G, 2 * G))]
                k = _exact_row(part[0], part[2].view(torch.bfloat16), orders[0])
                v = _exact_row(part[1], part[3].view(torch.bfloat16), orders[1])
            for m in range(h * group, (h + 1) * group):
                s = (x[r * n:(r + 1) * n, m] @ k.T) * state["scale"]
                out[r * n:(r + 1) * n, m] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v
    return out.reshape(-1, nh * hd)
