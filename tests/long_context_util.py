"""A plain Llama whose layers cache keys and values in 4 bits, or see a window and the first tokens only; and dense stand-ins of
the operators that do the same in the engine, for runs without a GPU."""
import math

import torch

import plain_llama
import standin_ops
from kv4_util import put, rounded, values_of


def held(x):
    """What 4 bits hold of keys or values [n, heads, dims]."""
    return values_of(*rounded(x)).to(x.dtype)


def attention(q, k, v, scale, window, first):
    n, nh, hd = q.shape
    k, v = (a.repeat_interleave(nh // a.shape[1], 1) for a in (k, v))
    s = torch.einsum("ihd,jhd->hij", q, k) * scale
    pos, key = torch.arange(n)[:, None], torch.arange(n)
    hidden = key > pos
    if window:
        hidden = hidden | ((key <= pos - window) & (key >= first))
    return torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(hidden, -math.inf), -1), v)


def forward_logits(cfg, w, tokens, kv4=False, window=None, first=0, act_round=None, key_round=None):
    """Logits [n, vocab] in 64 bits; ``key_round``: keys and values are rounded to this type before 4 bits, as a cache of the
    compute type would hold them."""
    rnd = plain_llama.bf16_rounding if act_round == "bfloat16" else plain_llama._no_rounding
    w = {k: v.double() for k, v in w.items()}
    nh, nkv, hd = plain_llama.sizes(cfg)
    inv = plain_llama.rope_inv_freq(hd, cfg.get("rope_theta", 10000.0), cfg.get("rope_scaling"))
    eps, n = cfg.get("rms_norm_eps", 1e-5), len(tokens)
    x = plain_llama.embed(w["model.embed_tokens.weight"], tokens)
    for i in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{i}."
        h = rnd(plain_llama.rms_norm(x, w[p + "input_layernorm.weight"], eps))
        q, k, v = (rnd(h @ w[p + f"self_attn.{name}_proj.weight"].T).view(n, -1, hd) for name in "qkv")
        q, k = (rnd(plain_llama.apply_rope(t, list(range(n)), inv)) for t in (q, k))
        if kv4:
            k, v = (held(t if key_round is None else t.to(key_round).double()) for t in (k, v))
        a = rnd(attention(q, k, v, 1.0 / math.sqrt(hd), window, first))
        x = x + rnd(a.reshape(n, nh * hd) @ w[p + "self_attn.o_proj.weight"].T)
        h = rnd(plain_llama.rms_norm(x, w[p + "post_attention_layernorm.weight"], eps))
        g, u = (rnd(h @ w[p + f"mlp.{name}_proj.weight"].T) for name in ("gate", "up"))
        x = x + rnd(rnd((g / (1.0 + torch.exp(-g))) * u) @ w[p + "mlp.down_proj.weight"].T)
    x = rnd(plain_llama.rms_norm(x, w["model.norm.weight"], eps))
    head = w["model.embed_tokens.weight"] if cfg.get("tie_word_embeddings", False) else w["lm_head.weight"]
    return x @ head.T


class Ops:
    """The stand-ins of the other kernels, and those of this file."""

    def __getattr__(self, name):
        return getattr(standin_ops, name)

    @staticmethod
    def _gather(ctx, cache, r, first, window, n, read):
        L, row = int(ctx.kv_len[r]), int(ctx.table_rows[r])
        lo = max(0, L - n - window + 1) if window else 0
        idx = torch.cat([torch.arange(min(first, lo) if window else 0), torch.arange(lo, L)])
        pages = cache.block_table[row, idx // cache.page_size].long()
        assert (pages >= 0).all(), "read of a page that is not held"
        return idx, *read(pages, idx % cache.page_size)

    def _attend(self, q, nh, nkv, hd, ctx, cache, scale, window, first, out, read):
        starts = ctx.q_start.tolist()
        for r in range(ctx.n_requests):
            a, n = starts[r], starts[r + 1] - starts[r]
            idx, K, V = self._gather(ctx, cache, r, first, window, n, read)
            K, V = (t.repeat_interleave(nh // nkv, 1) for t in (K.float(), V.float()))
            s = torch.einsum("ihd,jhd->hij", q[a:a + n, :nh * hd].float().view(n, nh, hd), K) * scale
            pos = torch.arange(int(ctx.kv_len[r]) - n, int(ctx.kv_len[r]))[:, None]
            hidden = idx[None] > pos
            if window:
                hidden = hidden | ((idx[None] <= pos - window) & (idx[None] >= first))
            o = torch.einsum("hij,jhd->ihd", torch.softmax(s.masked_fill(hidden, -math.inf), -1), V)
            out[a:a + n] = o.reshape(n, nh * hd).to(out.dtype)

    def paged_attention(self, qkv, nh, nkv, hd, ctx, cache, scale, window, out, first=0):
        self._attend(qkv, nh, nkv, hd, ctx, cache, scale, window, first, out, lambda p, o: (cache.k_pages[p, :, o], cache.v_pages[p, :, o]))

    def rope_store_attention(self, qkv, nh, nkv, hd, ctx, cache, inv_freq, rotary_dim, store, scale, window, out, first=0):
        standin_ops.rope_kv_store(qkv, nh, nkv, hd, ctx, cache, inv_freq, rotary_dim, store)
        self.paged_attention(qkv, nh, nkv, hd, ctx, cache, scale, window, out, first)

    def rope_kv4_store(self, qkv, nh, nkv, hd, ctx, cache, inv_freq, rotary_dim, q_out, store=True):
        T, half = qkv.shape[0], rotary_dim // 2
        x = qkv.view(T, nh + 2 * nkv, hd)
        a = ctx.positions.double()[:, None] * inv_freq.double()[None]
        c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
        lo, hi = x[:, :nh + nkv, :half].double(), x[:, :nh + nkv, half:rotary_dim].double()
        turned = torch.cat([lo * c - hi * s, lo * s + hi * c, x[:, :nh + nkv, rotary_dim:].double()], -1).to(qkv.dtype)
        q_out.copy_(turned[:, :nh].reshape(T, nh * hd))
        if store:
            (kc, ks), (vc, vs) = rounded(turned[:, nh:]), rounded(x[:, nh + nkv:])
            for t in range(T):
                put(cache.pages, cache.block_table[int(ctx.table_rows[int(ctx.token_req[t])])], cache.page_size, int(ctx.positions[t]),
                    kc[t], ks[t], vc[t], vs[t])

    def paged_attention_kv4(self, q, nh, nkv, hd, ctx, cache, scale, window, out, first=0):
        G, half = hd // 32, hd // 2
        d = torch.arange(hd)
        kb, vb = (d % 32 // 8 * G + d // 32) * 4 + d % 8 // 2, d % 16 // 2 * 2 * G + d // 16

        def read(pages, off):
            tile = cache.pages[pages, :, off // 16]                              # [n, kv heads, 18 hd]
            at = (off % 16)[:, None, None].expand(-1, nkv, 1)

            def part(base, width):
                return torch.gather(tile, 2, base + at * width + torch.arange(width)).contiguous()

            codes = [part(0, half)[..., kb] >> (4 * (d % 2)) & 15, part(8 * hd, half)[..., vb] >> (4 * (d % 2)) & 15]
            scales = [part(b, 2 * G).view(torch.bfloat16).double() for b in (16 * hd, 17 * hd)]
            return values_of(codes[0], scales[0]), values_of(codes[1], scales[1])

        self._attend(q, nh, nkv, hd, ctx, cache, scale, window, first, out, read)
