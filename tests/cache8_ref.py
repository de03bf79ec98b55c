"""Plain restatement of the cache held in 8 bits and of attention over it, for the tests."""
from __future__ import annotations

import math

import torch

BLOCK = 64
CODE = torch.float8_e4m3fn


def turned(x, table):
    """Rotate-half of f32 [rows, heads, dim] by [rows, dim] of cosines and sines, product by product."""
    half = x.shape[-1] // 2
    c, s = table[:, None, :half], table[:, None, half:]
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * c - b * s, a * s + b * c), dim=-1)


def project(qkv, positions, heads, kv_heads, dim, bias, rope):
    """(queries, keys, values) f16 of f16 rows at `positions`."""
    x = qkv.float()
    if bias is not None:
        x = x + bias
    x = x.unflatten(1, (heads + 2 * kv_heads, dim))
    qk = x[:, :heads + kv_heads]
    if rope is not None:
        qk = turned(qk, rope[positions])
    k, v = qk[:, heads:].half(), x[:, heads + kv_heads:].half()
    odd = ~v.isfinite().all(dim=-1)
    k = torch.where(k.isfinite(), k, math.nan)
    k[..., 0] = torch.where(odd, math.nan, k[..., 0])
    return qk[:, :heads].flatten(1).half(), k, torch.where(v.isfinite(), v, 0.0)


def block_codes(x):
    """f16 [BLOCK, dim] -> (codes as bytes, scale)."""
    y = x.double()
    finite = y[y.isfinite()]
    top = float(finite.abs().max()) if finite.numel() else 0.0
    e = 0
    if top > 0:
        e = math.ceil(math.log2(top / 448.0) - 1e-9)
        while top <= 448.0 * 2.0 ** (e - 1):
            e -= 1
        while top > 448.0 * 2.0 ** e:
            e += 1
    z = torch.where(y.isfinite(), y * 2.0 ** -e, math.nan).float()
    return z.to(CODE).view(torch.uint8), 2.0 ** e


class RefCache:
    """What every sequence holds, token by token, as f16 [kv_heads, length, dim]."""

    def __init__(self, seqs, kv_heads, dim):
        self.k = [torch.zeros((kv_heads, 0, dim), dtype=torch.float16, device="cuda") for _ in range(seqs)]
        self.v = [t.clone() for t in self.k]
        self.longest = [0] * seqs

    def append(self, seq, start, k, v):
        """k, v: [rows, kv_heads, dim] at position `start` (what was held from there on is dropped)."""
        self.k[seq] = torch.cat((self.k[seq][:, :start], k.transpose(0, 1)), dim=1)
        self.v[seq] = torch.cat((self.v[seq][:, :start], v.transpose(0, 1)), dim=1)
        self.longest[seq] = max(self.longest[seq], self.k[seq].shape[1])

    def check(self, cache):
        """The cache's bytes, where they say anything, are those of the tokens."""
        for seq, (k, v) in enumerate(zip(self.k, self.v)):
            n = k.shape[1]
            for x, codes, scale, tail in ((k, cache.k, cache.k_scale, cache.k_tail), (v, cache.v, cache.v_scale, cache.v_tail)):
                codes = codes.view(torch.uint8)
                for h in range(x.shape[0]):
                    for b in range(n // BLOCK):
                        want, s = block_codes(x[h, b * BLOCK:(b + 1) * BLOCK])
                        got = codes[seq, h, b * BLOCK:(b + 1) * BLOCK]
                        nan = (want & 0x7f) == 0x7f
                        assert torch.equal(got[~nan], want[~nan]) and bool(((got & 0x7f)[nan] == 0x7f).all()), (seq, h, b)
                        assert float(scale[seq, h, b]) == s, (seq, h, b)
                    for b in range(max(0, -(-self.longest[seq] // BLOCK) - 2), -(-n // BLOCK)):
                        want = x[h, b * BLOCK:(b + 1) * BLOCK].contiguous()
                        got = tail[seq, h, b % 2, :want.shape[0]]
                        assert torch.equal(got.isnan(), want.isnan()), (seq, h, b)
                        assert torch.equal(got.nan_to_num().view(torch.int16), want.nan_to_num().view(torch.int16)), (seq, h, b)

    def held(self, seq, length):
        """f64 [kv_heads, length, dim] of keys and values as attention sees them when the sequence has `length` tokens: full blocks rounded."""
        out = []
        for x in (self.k[seq][:, :length], self.v[seq][:, :length]):
            parts = []
            for b in range(length // BLOCK):
                per_head = []
                for h in range(x.shape[0]):
                    codes, s = block_codes(x[h, b * BLOCK:(b + 1) * BLOCK])
                    per_head.append(codes.view(CODE).double() * s)
                parts.append(torch.stack(per_head))
            parts.append(x[:, length // BLOCK * BLOCK:].double())
            out.append(torch.cat(parts, dim=1))
        return out


def attention(q, k, v, start, heads, scale, window):
    """(outputs, bound on a kernel's error) f64 [rows, heads * dim] of q f16 [rows, heads * dim] at positions start ..., over k, v f64 [kv_heads,
    length, dim].

    The bound: a weight enters the product with the values as FP16, off by half a step (2^-11 of itself, or 2^-25 of the largest weight times
    its value's scale, here over-estimated with the values' size); exponents are FP32, off by at most 2^-16 of a weight in all; sums are FP32
    (2^-18 of the sum of sizes); the result is FP16 (2^-11, 2^-25 next to zero).  A score is a sum of dim products in FP32, every partial sum
    of about the largest score's size at most and rounded by 2^-24 of itself, and then takes up to 8 more roundings: an exponent is off by
    that much, a weight and the sum of weights by as much of themselves each."""
    rows, group = q.shape[0], heads // k.shape[0]
    d = k.shape[2]
    x = torch.einsum("rhgd,hld->hgrl", q.double().unflatten(1, (k.shape[0], group, d)), k) * scale
    far = torch.arange(start, start + rows, device="cuda")[:, None] - torch.arange(k.shape[1], device="cuda")
    x = x.masked_fill(~((far >= 0) & (far < (window or 1 << 40))), -math.inf)
    p = torch.softmax(x, dim=-1)
    largest = x.masked_fill(x == -math.inf, 0.0).abs().nan_to_num().amax(dim=-1).permute(2, 0, 1).repeat_interleave(d, dim=2).flatten(1)
    out = torch.einsum("hgrl,hld->rhgd", p, v).flatten(1)
    size = torch.einsum("hgrl,hld->rhgd", p, v.abs()).flatten(1)
    seen = torch.einsum("hgrl,hld->rhgd", (p > 0).double(), v.abs()).flatten(1)
    top = p.amax(dim=-1).permute(2, 0, 1).repeat_interleave(d, dim=2).flatten(1)
    return out, 2.0 ** -11 * out.abs() + (2.0 ** -11 + 2.0 ** -15 + 2 * (d + 8) * 2.0 ** -24 * largest) * size + 2.0 ** -25 * top * seen + 2.0 ** -25


def attention_by_values(q, k, v, start, heads, scale, window):
    """As ``attention``, with a bound that shrinks with the values, however the sizes of blocks of them differ.

    Beside what the bound of ``attention`` says of scores, sums and the result: a weight times its values' unit enters the product as FP16, off by half a
    step: 2^-11 of itself, or 2^-25 where it is below 2^-14, when the largest one of the row so far lies at 2^7 at least, so 2^-32 of that one.  The unit of a
    full block is a power of two below 1/224 of its largest value ahead of the rounding to 4 bits, which takes 2^-4 of it at most; values of zeros have
    none.  That of the tail, which comes last, is one.  In its unit a value of a full block is at most 448."""
    rows, group, n = q.shape[0], heads // k.shape[0], k.shape[1]
    d = k.shape[2]
    x = torch.einsum("rhgd,hld->hgrl", q.double().unflatten(1, (k.shape[0], group, d)), k) * scale
    far = torch.arange(start, start + rows, device="cuda")[:, None] - torch.arange(n, device="cuda")
    x = x.masked_fill(~((far >= 0) & (far < (window or 1 << 40))), -math.inf)
    p = torch.softmax(x, dim=-1)
    wide = lambda t: t.permute(2, 0, 1).repeat_interleave(d, dim=2).flatten(1)  # noqa: E731
    largest = wide(x.masked_fill(x == -math.inf, 0.0).abs().amax(dim=-1))
    out = torch.einsum("hgrl,hld->rhgd", p, v).flatten(1)
    size = torch.einsum("hgrl,hld->rhgd", p, v.abs()).flatten(1)
    top = torch.stack([v[:, b:b + BLOCK].abs().amax(dim=(1, 2)) for b in range(0, n, BLOCK)], dim=1).repeat_interleave(BLOCK, dim=1)[:, :n]
    unit = top / (224 * (1 - 2.0 ** -4))
    full = n // BLOCK * BLOCK
    small = (p[..., :full] * unit[:, None, None, :full]).amax(dim=-1) * 448.0 * full if full else torch.zeros_like(p[..., 0])
    if full < n:
        unit[:, full:] = 1.0
        small = small + (p * unit[:, None, None]).amax(dim=-1) * top[:, None, None, -1] * (n - full)
    return out, 2.0 ** -11 * out.abs() + (2.0 ** -11 + 2.0 ** -15 + 2 * (d + 8) * 2.0 ** -24 * largest) * size + 2.0 ** -32 * wide(small) + 2.0 ** -25
