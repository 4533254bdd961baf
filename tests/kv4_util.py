"""A 4-bit cache of keys and values restated with tensor arithmetic: rounding, the layout of a page, attention in 64 bits."""
import math
import types

import numpy as np
import torch

GROUP = 32


def scale_of(largest):
    """A seventh of it in 32-bit, rounded to 5 significant bits (ties to even); none below 2^-100."""
    part, power = np.frexp(np.float32(largest.double().cpu().numpy() / 7.0).astype(np.float64))
    s = torch.from_numpy(np.asarray(np.ldexp(np.rint(part * 32), power - 5)))
    return torch.where(largest.cpu() < 2.0 ** -100, torch.zeros_like(s), s).to(largest.device)


def rounded(x):
    """(codes 0..15, scales in 64-bit) of x [..., dims]; a group with a number that is not finite has a scale that is none."""
    g = x.double().unflatten(-1, (-1, GROUP))
    fine = torch.isfinite(g).all(-1, keepdim=True)
    g = torch.where(fine, g, torch.zeros_like(g))
    s = scale_of(g.abs().amax(-1, keepdim=True))
    n = torch.round(g / torch.where(s > 0, s, torch.ones_like(s))).clamp(-7, 7)
    n = torch.where(s > 0, n, torch.zeros_like(n))
    return (n + 8).to(torch.uint8).flatten(-2), torch.where(fine, s, torch.full_like(s, math.nan)).squeeze(-1)


def values_of(codes, scales):
    return ((codes.double() - 8).unflatten(-1, (-1, GROUP)) * scales.unsqueeze(-1)).flatten(-2)


def row_bytes(codes, value):
    """The bytes of rows of codes [..., dims], in the order that the cache keeps keys' or values' rows."""
    hd = codes.shape[-1]
    G = hd // GROUP
    out = torch.zeros(codes.shape[:-1] + (hd // 2,), dtype=torch.uint8, device=codes.device)
    for d in range(hd):
        if value:
            byte, shift = (d % 16 // 2) * 2 * G + d // 16, 4 * (d % 2)
        else:
            byte, shift = ((d % 32 // 8) * G + d // 32) * 4 + d % 8 // 2, 4 * (d % 2)
        out[..., byte] |= codes[..., d] << shift
    return out


def put(pages, table_row, page_size, pos, kc, ks, vc, vs):
    """Write codes and scales [kv heads, ...] of the token at ``pos`` of the request whose pages are ``table_row``."""
    hd = kc.shape[-1]
    tile = pages[int(table_row[pos // page_size]), :, pos % page_size // 16]        # [kv heads, 18 hd]
    r, G = pos % 16, hd // GROUP
    tile[:, r * hd // 2:(r + 1) * hd // 2] = row_bytes(kc, False)
    tile[:, 8 * hd + r * hd // 2:8 * hd + (r + 1) * hd // 2] = row_bytes(vc, True)
    for base, s in ((16 * hd, ks), (17 * hd, vs)):
        tile[:, base + r * 2 * G:base + (r + 1) * 2 * G] = s.to(torch.bfloat16).contiguous().view(torch.uint8)


def step(q_lens, kv_lens, rows=None, fixed=False):
    """A step's metadata as the engine's kernels get it."""
    q, kv = np.array(q_lens, dtype=np.int32), np.array(kv_lens, dtype=np.int32)
    R = len(q_lens)
    rows = np.arange(R, dtype=np.int32) if rows is None else np.array(rows, dtype=np.int32)
    start = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
    pos = np.concatenate([np.arange(L - n, L) for n, L in zip(q_lens, kv_lens)]).astype(np.int32)

    def dev(a):
        return torch.from_numpy(np.ascontiguousarray(a)).cuda()

    return types.SimpleNamespace(
        n_tokens=int(q.sum()), n_requests=R, max_q_len=int(q.max()), max_kv_len=int(kv.max()), h_q_len=q, h_kv_len=kv,
        h_q_start=start, h_table_rows=rows, positions=dev(pos), token_req=dev(np.repeat(np.arange(R, dtype=np.int32), q)),
        q_start=dev(start), kv_len=dev(kv), table_rows=dev(rows), fixed_launch=fixed)


def attention(q, K, V, L, scale, window, first, steps):
    """64-bit attention of q [n, heads, hd] (the last n of L positions) over K, V [L, kv heads, hd]: the result, and the sums of
    weights times the values' magnitudes and times their ``steps`` [L, kv heads, hd] (the scale of each value's group)."""
    n, nh, hd = q.shape
    group = nh // K.shape[1]
    K, V, steps = (x.double().repeat_interleave(group, 1) for x in (K, V, steps))
    s = torch.einsum("ihd,jhd->hij", q.double(), K) * scale
    pos, key = torch.arange(L - n, L, device=q.device)[:, None], torch.arange(L, device=q.device)
    hidden = key > pos
    if window:
        hidden = hidden | ((key <= pos - window) & (key >= first))
    w = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
    live = torch.where(hidden, torch.zeros_like(w), w)
    V0, hide = torch.nan_to_num(V, nan=0.0), hidden.all(0)
    V0 = torch.where(hide[:, None, None], torch.zeros_like(V0), V0)
    return tuple(torch.einsum("hij,jhd->ihd", live, x) for x in (V0, V0.abs(), torch.nan_to_num(steps, nan=0.0)))
