"""The generation operators together, as a decoder uses them: a Llama-style
model of this library's own ops with its keys and values in the paged 4-bit
cache, prompts of mixed lengths taken in at once, then token by token."""
import ctypes as C

import numpy as np
import pytest

from gollama_b200 import synthetic as syn
from gollama_b200._lib import KVBatchC, KVCacheC
from tests import generation_ref as ref
from tests.helpers import rel_fro

pytestmark = pytest.mark.gpu

SHAPE = syn.TINY_LLAMA_MODE
EPS, PAGE, PAGES, MAX = SHAPE.norm_eps, 16, 24, 64


class Model:
    """Weights on the device; one forward of new tokens over the cache."""

    def __init__(self, ctx, shape, seed):
        self.ctx, self.shape, self.np = ctx, shape, {}
        flat, at = syn.init_params(shape, seed, std=0.08), 0
        for name, (r, c) in syn.param_shapes(shape):
            self.np[name] = flat[at:at + r * c].reshape(r, c)
            at += r * c
        self.np["OutputNorm"] = self.np["OutputNorm"] + np.float32(0.25)
        self.dev = {k: ctx.from_numpy(v) for k, v in self.np.items()}
        for l in range(shape.layers):
            n = self.np
            self.dev[f"L{l}.QKV"] = ctx.from_numpy(np.concatenate([n[f"L{l}.WQ"], n[f"L{l}.WK"], n[f"L{l}.WV"]]))
            self.dev[f"L{l}.GU"] = ctx.from_numpy(np.concatenate([n[f"L{l}.WGate"], n[f"L{l}.WUp"]]))
        hd = shape.head_dim
        self.cos, self.sin = np.zeros((MAX, hd // 2), np.float32), np.zeros((MAX, hd // 2), np.float32)
        ctx.lib.glc_rope_table(hd, MAX, C.c_float(shape.rope_theta), self.cos.ctypes.data_as(C.c_void_p), self.sin.ctypes.data_as(C.c_void_p))
        self.dcos, self.dsin = ctx.from_numpy(self.cos), ctx.from_numpy(self.sin)
        self.bytes = C.c_size_t()
        cache = KVCacheC(num_pages=PAGES, page_size=PAGE, num_kv_heads=shape.kv_heads, head_dim=hd)
        assert ctx.lib.glc_kv_cache_bytes(C.byref(cache), C.byref(self.bytes)) == 0
        self.pools = [(ctx.zeros((self.bytes.value,), np.uint8), ctx.zeros((self.bytes.value,), np.uint8)) for _ in range(shape.layers)]
        self.caches = [KVCacheC(k=k.addr, v=v.addr, num_pages=PAGES, page_size=PAGE, num_kv_heads=shape.kv_heads, head_dim=hd)
                       for k, v in self.pools]

    def forward(self, tokens, batch):
        """Logits [T][vocab] on the device."""
        ctx, s, T = self.ctx, self.shape, len(tokens)
        d, H, Hkv, hd, F = s.hidden, s.heads, s.kv_heads, s.head_dim, s.inter
        w = (H + 2 * Hkv) * hd
        ids, x, y, rms = ctx.from_numpy(np.asarray(tokens, np.int64)), ctx.empty((T, d)), ctx.empty((T, d)), ctx.empty((T,))
        qkv, o, gu, h = ctx.empty((T, w)), ctx.zeros((T, H * hd)), ctx.empty((T, 2 * F)), ctx.empty((T, F))
        ctx.call("glc_embed_fwd", ids.ptr, self.dev["TokenEmbed"].ptr, None, x.ptr, T, T, d, s.vocab)
        for l in range(s.layers):
            p = lambda n: self.dev[f"L{l}.{n}"].ptr  # noqa: E731
            ctx.call("glc_rmsnorm_fwd", x.ptr, p("AttnNorm"), y.ptr, rms.ptr, T, d, C.c_float(EPS), 0)
            ctx.call("glc_linear_fwd", y.ptr, p("QKV"), qkv.ptr, T, d, w, None)
            a, cache = qkv.addr, C.byref(self.caches[l])
            ctx.call("glc_kv_append", cache, C.byref(batch), a, w, a, w, H, a + 4 * H * hd, w, a + 4 * (H + Hkv) * hd, w,
                     self.dcos.ptr, self.dsin.ptr, MAX)
            ctx.call("glc_attention_kv", cache, C.byref(batch), a, w, H, o.ptr, H * hd, None)
            ctx.call("glc_linear_fwd", o.ptr, p("WO"), x.ptr, T, d, d, x.ptr)
            ctx.call("glc_rmsnorm_fwd", x.ptr, p("FFNNorm"), y.ptr, rms.ptr, T, d, C.c_float(EPS), 0)
            ctx.call("glc_linear_fwd_swiglu", y.ptr, p("GU"), gu.ptr, h.ptr, T, d, F, 0)
            ctx.call("glc_linear_fwd", h.ptr, p("WDown"), x.ptr, T, F, d, x.ptr)
        logits = ctx.empty((T, s.vocab))
        ctx.call("glc_rmsnorm_fwd", x.ptr, self.dev["OutputNorm"].ptr, y.ptr, rms.ptr, T, d, C.c_float(EPS), 0)
        ctx.call("glc_linear_fwd", y.ptr, self.dev["TokenEmbed"].ptr, logits.ptr, T, d, s.vocab, None)
        ctx.held = (ids, x, y, rms, qkv, o, gu, h)
        return logits

    def stored(self, l, table, length):
        """Keys and values of a sequence as the cache holds them."""
        ctx, s = self.ctx, self.shape
        w = s.kv_heads * s.head_dim
        held = [ctx.from_numpy(np.asarray(x, np.int32)) for x in ([table], [length], [0, length])]
        b = KVBatchC(page_table=held[0].addr, lens=held[1].addr, starts=held[2].addr, num_seqs=1, max_pages=len(table), num_rows=length)
        k, v = ctx.empty((length, w)), ctx.empty((length, w))
        ctx.call("glc_kv_read", C.byref(self.caches[l]), C.byref(b), k.ptr, w, v.ptr, w)
        ctx.sync()
        return [x.numpy().astype(np.float64).reshape(length, s.kv_heads, s.head_dim) for x in (k, v)]

    def exact(self, tokens, table):
        """Logits of a whole sequence in 64 bits, attending to what the cache holds."""
        s, n = self.shape, {k: v.astype(np.float64) for k, v in self.np.items()}
        T, hd = len(tokens), s.head_dim
        norm = lambda z, w: z / np.sqrt((z * z).mean(1, keepdims=True) + EPS) * w  # noqa: E731
        x = n["TokenEmbed"][tokens]
        for l in range(s.layers):
            y = norm(x, n[f"L{l}.AttnNorm"])
            q = ref.rotate((y @ n[f"L{l}.WQ"].T).reshape(T, s.heads, hd), self.cos.astype(np.float64), self.sin.astype(np.float64), np.arange(T))
            k, v = self.stored(l, table, T)
            own = ref.rotate((y @ n[f"L{l}.WK"].T).reshape(T, s.kv_heads, hd), self.cos.astype(np.float64), self.sin.astype(np.float64), np.arange(T))
            assert rel_fro(k, own) < 0.12 and rel_fro(v, (y @ n[f"L{l}.WV"].T).reshape(v.shape)) < 0.12  # 4 bits of them
            o = np.zeros((T, s.heads, hd))
            for h in range(s.heads):
                kk, vv = k[:, h * s.kv_heads // s.heads], v[:, h * s.kv_heads // s.heads]
                a = np.where(np.tri(T, dtype=bool), q[:, h] @ kk.T / np.sqrt(hd), -np.inf)
                a = np.exp(a - a.max(1, keepdims=True))
                o[:, h] = a @ vv / a.sum(1, keepdims=True)
            x = x + o.reshape(T, -1) @ n[f"L{l}.WO"].T
            y = norm(x, n[f"L{l}.FFNNorm"])
            g = y @ n[f"L{l}.WGate"].T
            x = x + (g / (1 + np.exp(-g)) * (y @ n[f"L{l}.WUp"].T)) @ n[f"L{l}.WDown"].T
        return norm(x, n["OutputNorm"]) @ n["TokenEmbed"].T


def batch_of(ctx, table, lens, starts):
    held = [ctx.from_numpy(np.ascontiguousarray(x, np.int32)) for x in (table, lens)]
    held.append(None if starts is None else ctx.from_numpy(np.ascontiguousarray(starts, np.int32)))
    b = KVBatchC(page_table=held[0].addr, lens=held[1].addr, starts=0 if starts is None else held[2].addr, num_seqs=len(lens),
                 max_pages=table.shape[1], num_rows=len(lens) if starts is None else int(starts[-1]))
    b.held = held
    return b


# the linear layers round their operands to TF32: 2^-11 of each, of either sign, over
# ~15 of them in a row 15^1/2 2^-11 (1.9e-3) in all, three of which are taken
LOGITS = 3 * 15**0.5 * 2.0**-11


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_prompts_then_tokens(ctx, temperature):
    r = np.random.default_rng(31)
    model = Model(ctx, SHAPE, 5)
    seqs = [list(map(int, r.integers(0, SHAPE.vocab, n))) for n in (5, 1, 18)]
    B = len(seqs)
    table = r.permutation(PAGES)[: B * 4].reshape(B, 4).astype(np.int32)
    # the prompts at once
    starts = np.concatenate([[0], np.cumsum([len(s) for s in seqs])])
    logits = model.forward(sum(seqs, []), batch_of(ctx, table, [len(s) for s in seqs], starts))
    ctx.sync()
    got = logits.numpy()
    for b, s in enumerate(seqs):
        assert rel_fro(got[starts[b]:starts[b + 1]], model.exact(s, table[b])) < LOGITS
    last = got[starts[1:] - 1]
    for step in range(20):  # into the second and third pages
        u = r.random(B, dtype=np.float32)
        d = [ctx.from_numpy(x) for x in (last, np.full(B, temperature, np.float32), np.full(B, 30, np.int32), np.full(B, 0.9, np.float32), u)]
        tok, logp = ctx.empty((B,), np.int64), ctx.empty((B,))
        ctx.call("glc_sample", d[0].ptr, SHAPE.vocab, B, SHAPE.vocab, d[1].ptr, d[2].ptr, d[3].ptr, None, d[4].ptr, tok.ptr, logp.ptr)
        ctx.sync()
        for b in range(B):
            ids, w = ref.kept_tokens(last[b], np.float32(temperature), 30, np.float32(0.9), 0.0)
            upto = np.cumsum(w) / w.sum()
            at = min(int((upto <= float(u[b])).sum()), len(ids) - 1)
            near = [at] + [i for i in (at - 1, at + 1) if 0 <= i < len(ids) and abs(upto[min(i, at)] - float(u[b])) < 1e-6]
            assert tok.numpy()[b] in ids[near]
            seqs[b].append(int(tok.numpy()[b]))
        logits = model.forward([s[-1] for s in seqs], batch_of(ctx, table, [len(s) for s in seqs], None))
        ctx.sync()
        last = logits.numpy()
        if step in (0, 1, 10, 19):
            for b, s in enumerate(seqs):
                assert rel_fro(last[b], model.exact(s, table[b])[-1]) < LOGITS


def test_a_prompt_in_pieces_is_the_prompt(ctx):
    """A prompt in one call, in chunks, and token by token: the same cache, but for
    codes at whose edge the linear layers' kernels for few and for many rows round to
    either side (one in 10^4 would need products that differ by 10^-5), and the same
    logits."""
    r = np.random.default_rng(32)
    tokens = list(map(int, r.integers(0, SHAPE.vocab, 37)))
    table = np.array([[3, 0, 7]], np.int32)
    out, held = [], []
    for cuts in ([37], [16, 37], [5, 6, 30, 37], list(range(1, 38))):
        model = Model(ctx, SHAPE, 6)
        done, last = 0, None
        for end in cuts:
            last = model.forward(tokens[done:end], batch_of(ctx, table, [end], [0, end - done]))
            done = end
        ctx.sync()
        out.append(last.numpy()[-1])
        held.append([np.concatenate([p.numpy() for p in pools]) for pools in model.pools])
    for o, h in zip(out[1:], held[1:]):
        same = np.mean([np.mean(a == b) for a, b in zip(h, held[0])])
        assert same > 0.999, same
        assert rel_fro(o, out[0]) < LOGITS
