"""GPU tests of the cache held in 8 bits: the append against its definition bit for bit, attention against plain attention in 64 bits."""
import math
import zlib

import pytest
import torch

import cache8_ref as ref
from tensorwarp_b200 import _lib, cache8

pytestmark = pytest.mark.gpu
HEADS = [(28, 4, 128), (8, 8, 64), (5, 1, 128), (40, 8, 64), (16, 4, 128)]


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def gen(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def poisoned(seqs, capacity, kv_heads, dim):
    """An empty cache whose every place holds NaN: what is not filled must not be looked at."""
    c = cache8.Cache8.empty(seqs, capacity, kv_heads, dim)
    for t in (c.k, c.v):
        t.view(torch.uint8).fill_(0x7f)
    for t in (c.k_scale, c.v_scale, c.k_tail, c.v_tail):
        t.fill_(math.nan)
    return c


class Batch:
    """A cache, its restatement, and where every sequence stands."""

    def __init__(self, seqs, capacity, heads, kv_heads, dim, seed=0, bias=True, rope=True, make=None):
        self.heads, self.kv_heads, self.dim, self.seqs = heads, kv_heads, dim, seqs
        self.cache = poisoned(seqs, capacity, kv_heads, dim)
        self.held = ref.RefCache(seqs, kv_heads, dim)
        self.gen = gen("batch", seed)
        self.width = (heads + 2 * kv_heads) * dim
        self.bias = 0.5 * torch.randn(self.width, generator=self.gen, device="cuda") if bias else None
        self.rope = cache8.rope_table(self.cache.capacity, dim, 1e4) if rope else None
        self.make = make or (lambda rows: torch.randn((rows, self.width), generator=self.gen, device="cuda") * torch.exp(
            torch.randn((1, self.width), generator=gen("channel", seed), device="cuda")))

    def append(self, starts, counts, pad=0, **kw):
        """One call; returns (queries of the call's rows, row_start, max_rows)."""
        row_start = [0]
        for n in counts:
            row_start.append(row_start[-1] + n)
        total = row_start[-1] + pad
        qkv = self.make(total).half()
        q = torch.full((total, self.heads * self.dim), 7.0, dtype=torch.float16, device="cuda")
        most = max(max(counts), 1)
        cache8.append(self.cache, qkv, q, ints(starts), num_heads=self.heads, row_start=ints(row_start), max_rows=most, bias=self.bias, rope=self.rope, **kw)
        for s, (start, n) in enumerate(zip(starts, counts)):
            rows = slice(row_start[s], row_start[s] + n)
            if start < 0 or n == 0:
                assert bool((q[rows] == 7.0).all())
                continue
            fit = min(n, self.cache.capacity - start)
            positions = torch.arange(start, start + fit, device="cuda")
            qs, k, v = ref.project(qkv[rows][:fit], positions, self.heads, self.kv_heads, self.dim, self.bias, self.rope)
            assert torch.equal(q[rows][:fit], qs) and bool((q[rows][fit:] == 7.0).all())
            self.held.append(s, start, k, v)
        assert bool((q[row_start[-1]:] == 7.0).all())
        return q, row_start, most

    def attend(self, starts, counts, q=None, window=0, scale=None, pad=0, ld=None, **kw):
        row_start = [0]
        for n in counts:
            row_start.append(row_start[-1] + n)
        total, width = row_start[-1] + pad, self.heads * self.dim
        if q is None:
            q = 2 * torch.randn((total, width), generator=self.gen, device="cuda").half()
        out = torch.full((total, ld or width), 7.0, dtype=torch.float16, device="cuda")
        most = max(max(counts), 1)
        scale = scale or 1 / math.sqrt(self.dim)
        cache8.attention(self.cache, q[:total], out[:, :width], ints(starts), num_heads=self.heads, row_start=ints(row_start), max_rows=most, scale=scale,
                         window=window, **kw)
        torch.cuda.synchronize()
        assert _lib.lib().twm_device_error(None, _lib.C.byref(_lib.C.c_uint())) == 0
        assert bool((out[row_start[-1]:] == 7.0).all()) and bool((out[:, width:] == 7.0).all())
        for s, (start, n) in enumerate(zip(starts, counts)):
            got = out[row_start[s]:row_start[s] + n, :width].double()
            if start < 0:
                assert bool((got == 0).all())
                continue
            if n == 0:
                continue
            k, v = self.held.held(s, start + n)
            want, off = ref.attention(q[row_start[s]:row_start[s] + n], k, v, start, self.heads, scale, window)
            worst = ((got - want).abs() / off).max()
            assert bool(worst <= 1), (s, start, n, float(worst))
        return out


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("portions", [[1] * 3, [64], [63, 1, 1], [65], [200], [60, 10, 70, 1, 1, 126], [1, 300], [100, 200, 129, 3], [640]])
def test_append(heads, kv_heads, dim, portions):
    b = Batch(1, 700, heads, kv_heads, dim, seed=len(portions))
    at = 0
    for n in portions:
        b.append([at], [n])
        at += n
        b.held.check(b.cache)


def test_append_ragged_with_rows_left_out():
    """Sequences without rows, out of the call, at the capacity and past it; rows of padding."""
    b = Batch(6, 256, 8, 2, 128)
    b.append([0, 0, -1, 0, 0, 0], [130, 0, 5, 1, 64, 250], pad=4)
    b.held.check(b.cache)
    b.append([130, 0, 0, 1, 64, 250], [2, 3, 70, 0, 150, 20], pad=1)
    b.held.check(b.cache)
    b.append([132, 3, 70, 1, 214, 256], [1, 1, 1, 1, 1, 1])
    b.held.check(b.cache)


@pytest.mark.parametrize("bias,rope", [(False, False), (True, False), (False, True)])
def test_append_without_bias_or_rotation(bias, rope):
    b = Batch(2, 192, 4, 2, 64, bias=bias, rope=rope)
    b.append([0, 0], [100, 64])
    b.append([100, 64], [1, 70])
    b.held.check(b.cache)


def test_one_row_a_sequence_without_row_start():
    b = Batch(3, 128, 8, 2, 128)
    starts = [0, 63, 64]
    b.append([0, 0, 0], [0, 63, 64])
    qkv = b.make(3).half()
    q = torch.zeros((3, 8 * 128), dtype=torch.float16, device="cuda")
    cache8.append(b.cache, qkv, q, ints(starts), num_heads=8, bias=b.bias, rope=b.rope)
    for s, start in enumerate(starts):
        qs, k, v = ref.project(qkv[s:s + 1], torch.tensor([start], device="cuda"), 8, 2, 128, b.bias, b.rope)
        assert torch.equal(q[s:s + 1], qs)
        b.held.append(s, start, k, v)
    b.held.check(b.cache)
    out = torch.zeros_like(q)
    cache8.attention(b.cache, q, out, ints(starts), num_heads=8)
    for s, start in enumerate(starts):
        want, off = ref.attention(q[s:s + 1], *b.held.held(s, start + 1), start, 8, 1 / math.sqrt(128), 0)
        assert bool(((out[s:s + 1].double() - want).abs() <= off).all())


def test_portions_do_not_matter():
    """The same tokens in other portions leave the same bytes."""
    qkv = torch.randn((1, 500, 8 * 128), generator=gen("p"), device="cuda").half()
    rope, seen = cache8.rope_table(512, 128, 1e6), []
    for portions in ([500], [1] * 500, [63, 2, 64, 65, 6, 300], [250, 250]):
        cache, at = cache8.Cache8.empty(1, 512, 2, 128), 0
        for n in portions:
            q = torch.zeros((n, 4 * 128), dtype=torch.float16, device="cuda")
            cache8.append(cache, qkv[0, at:at + n], q, ints([at]), num_heads=4, row_start=ints([0, n]), max_rows=n, rope=rope)
            at += n
        for tail in (cache.k_tail, cache.v_tail):
            tail[:, :, 500 // 64 % 2, 500 % 64:] = 0                # places that hold no token of the sequence
        seen.append([t.view(torch.uint8).clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.k_tail, cache.v_tail)])
    for other in seen[1:]:
        for x, y in zip(seen[0], other):
            assert torch.equal(x, y)


def test_cut_back_and_appended_again():
    """A sequence goes back as far as the block before its last, into and over the border of a block."""
    b = Batch(1, 512, 4, 2, 64)
    b.append([0], [300])
    for start, n in ((256, 3), (200, 5), (192, 64), (192, 70), (255, 2), (200, 130)):
        b.append([start], [n])
        b.held.check(b.cache)
        b.attend([start], [n])


@pytest.mark.parametrize("fill", ["zeros", "small", "large", "odd"])
def test_values_at_the_ends_of_the_range(fill):
    """Blocks of zeros, of the smallest and largest FP16 numbers, and with infinities and NaN."""
    def make(rows):
        x = torch.randn((rows, 3 * 64), generator=gen(fill), device="cuda")
        if fill == "zeros":
            return x * 0
        if fill == "small":
            return x * 2.0 ** -23
        if fill == "large":
            return (x * 3e4).clamp(-65504, 65504)
        x[3, 70], x[70, 80], x[5, 150], x[64, 130] = math.inf, math.nan, -math.inf, math.nan
        return x
    b = Batch(1, 256, 1, 1, 64, bias=False, rope=False, make=make)
    b.append([0], [200])
    b.held.check(b.cache)


def test_amax_on_the_border_of_a_scale():
    """448 * 2^e is the largest value of scale 2^e, the next FP16 number takes the next scale."""
    for e in range(-20, 8):
        for value, want in ((448.0 * 2.0 ** e, e), (448.5 * 2.0 ** e, e + 1), (256.0 * 2.0 ** e, e), (224.0 * 2.0 ** e, e - 1)):
            if value > 65504 or float(torch.tensor(value).half()) != value:
                continue
            cache = cache8.Cache8.empty(1, 64, 1, 64)
            qkv = torch.zeros((64, 192), dtype=torch.float16, device="cuda")
            qkv[17, 64 + 5] = -value
            q = torch.zeros((64, 64), dtype=torch.float16, device="cuda")
            cache8.append(cache, qkv, q, ints([0]), num_heads=1, row_start=ints([0, 64]), max_rows=64)
            assert float(cache.k_scale[0, 0, 0]) == 2.0 ** want and float(cache.v_scale[0, 0, 0]) == 1.0


# ---------------------------------------------------------------------------------------------------------- attention --

@pytest.mark.parametrize("heads,kv_heads,dim", HEADS + [(71, 1, 64), (12, 2, 128), (33, 1, 128)])
@pytest.mark.parametrize("window", [0, 50])
def test_single_tokens(heads, kv_heads, dim, window):
    lengths = [1, 2, 17, 63, 64, 65, 127, 128, 129, 300, 1025]
    b = Batch(len(lengths), 1088, heads, kv_heads, dim)
    b.append([0] * len(lengths), lengths)
    b.attend([n - 1 for n in lengths], [1] * len(lengths), window=window)


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS + [(33, 1, 64)])
@pytest.mark.parametrize("window", [0, 1, 64, 100])
@pytest.mark.parametrize("rows", [2, 4, 7, 33, 200])
def test_rows_of_a_portion(heads, kv_heads, dim, window, rows):
    starts = [0, 1, 63, 64, 100, 500]
    counts = [rows, rows, max(1, rows // 2), rows, 1, rows]
    b = Batch(len(starts), 768, heads, kv_heads, dim)
    b.append([0] * len(starts), [s + n for s, n in zip(starts, counts)])
    b.attend(starts, counts, window=window, pad=2)


def test_ragged_batch_with_sequences_left_out():
    b = Batch(7, 512, 8, 2, 128)
    lengths = [400, 0, 64, 30, 512, 1, 129]
    b.append([0] * 7, lengths)
    for counts in ([1, 0, 1, 1, 1, 1, 1], [70, 0, 3, 30, 300, 1, 0]):
        starts = [n - c for n, c in zip(lengths, counts)]
        starts[2] = -1
        b.attend(starts, counts, pad=5)


def test_strides_and_repeat():
    """Rows inside wider buffers; the same call gives the same bits."""
    b = Batch(2, 256, 8, 2, 64)
    b.append([0, 0], [200, 130])
    for counts in ([1, 1], [40, 60]):
        wide = 2 * torch.randn((sum(counts), 8 * 64 + 24), generator=b.gen, device="cuda").half()
        starts = [200 - counts[0], 130 - counts[1]]
        x = b.attend(starts, counts, q=wide[:, 8:8 + 512], ld=8 * 64 + 16)
        assert torch.equal(x, b.attend(starts, counts, q=wide[:, 8:8 + 512], ld=8 * 64 + 16))


@pytest.mark.parametrize("rows", [1, 40])
def test_blocks_of_very_different_scale(rows):
    """Values of 2^15 and 2^-18 in neighbouring blocks, keys of 2^8 and 2^-8: neither scale drowns the other."""
    def make(n):
        x = torch.randn((n, 3 * 128), generator=gen("s", n), device="cuda")
        big = (torch.arange(n, device="cuda") // 64 % 2 == 0)[:, None]
        x[:, 128:256] *= torch.where(big, 2.0 ** 2, 2.0 ** -8)
        x[:, 256:] *= torch.where(big, 2.0 ** -18, 2.0 ** 12)
        return x
    b = Batch(1, 512, 1, 1, 128, bias=False, rope=False, make=make)
    b.append([0], [460])
    b.attend([460 - rows], [rows])
    b.attend([460 - rows], [rows], scale=4.0)


@pytest.mark.parametrize("rows", [1, 40])
def test_sharp_scores(rows):
    """Scores of thousands, growing and falling along the keys: the running maximum moves by all of it."""
    for slope in (3.0, -3.0):
        def make(n):
            x = torch.randn((n, 3 * 64), generator=gen("t", n), device="cuda")
            x[:, 64] += slope * torch.arange(n, device="cuda")
            return x
        b = Batch(1, 640, 1, 1, 64, bias=False, rope=False, make=make)
        b.append([0], [600])
        q = torch.randn((rows, 64), generator=gen("u"), device="cuda").half()
        q[:, 0] = 4.0
        b.attend([600 - rows], [rows], q=q, scale=1.0)


@pytest.mark.parametrize("column", [64 + 9, 128 + 9])
@pytest.mark.parametrize("rows", [1, 3, 70])
def test_tokens_that_are_no_numbers(rows, column):
    """A key or value that is infinite or NaN makes the rows that see it NaN, and no others, in a full block and in the tail."""
    for token, length in ((100, 150), (100, 128), (140, 150), (100, 101)):
        def make(n):
            x = torch.randn((n, 4 * 64), generator=gen("x", n), device="cuda")
            x[token, 64 + column] = math.inf if rows == 3 else math.nan
            return x
        b = Batch(1, 256, 2, 1, 64, bias=False, rope=False, make=make)
        b.append([0], [length])
        q = torch.randn((rows, 128), generator=b.gen, device="cuda").half()
        for window in (0, 5, 49):
            out = torch.zeros_like(q)
            cache8.attention(b.cache, q, out, ints([length - rows]), num_heads=2, row_start=ints([0, rows]), max_rows=rows, window=window)
            p = torch.arange(length - rows, length, device="cuda")
            sees = (p >= token) & (p - token < (window or 1 << 30))
            assert torch.equal(out.isnan(), sees[:, None].expand(rows, 128)), (token, length, window)


def test_far_places():
    """A cache whose places pass 2^32 bytes."""
    cap = (1 << 25) + 64
    cache = cache8.Cache8.empty(1, cap, 2, 128)
    start = cap - 70
    q = torch.randn((1, 512), generator=gen("far"), device="cuda").half()
    held = ref.RefCache(1, 2, 128)
    at = cap - 256
    for n in (64, 64, 58):                        # whole blocks at the far end
        qkv = torch.randn((n, 1024), generator=gen("far", at), device="cuda").half()
        out = torch.zeros((n, 512), dtype=torch.float16, device="cuda")
        cache8.append(cache, qkv, out, ints([at]), num_heads=4, row_start=ints([0, n]), max_rows=n)
        _, k, v = ref.project(qkv, None, 4, 2, 128, None, None)
        held.append(0, held.k[0].shape[1], k, v)
        at += n
    out = torch.zeros_like(q)
    cache8.attention(cache, q, out, ints([at - 1]), num_heads=4, window=186)
    k, v = held.held(0, 186)
    want, off = ref.attention(q, k, v, 185, 4, 1 / math.sqrt(128), 186)
    assert bool(((out.double() - want).abs() <= off).all())


@pytest.mark.parametrize("heads,kv_heads,dim,rows", [(40, 8, 128, 1), (16, 8, 64, 4), (28, 4, 128, 5), (16, 4, 128, 40)])
def test_long_batches_give_the_same_bits_again(heads, kv_heads, dim, rows):
    """Stages are used over and over, tiles begin and end anywhere in a CTA's run: a hundred calls, one result."""
    seqs, cap = 64, 4096
    cache = cache8.Cache8.empty(seqs, cap, kv_heads, dim)
    g = gen("long", heads, rows)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).copy_(torch.randint(0, 0x70, t.shape, generator=g, device="cuda", dtype=torch.uint8))
    for t in (cache.k_tail, cache.v_tail):
        t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
    cache.k_scale.fill_(2.0 ** -7), cache.v_scale.fill_(2.0 ** -6)
    q = torch.randn((seqs * rows, heads * dim), generator=g, device="cuda").half()
    start = torch.randint(0, cap - rows, (seqs,), generator=g, device="cuda", dtype=torch.int32)
    row_start = ints([rows * s for s in range(seqs + 1)])
    ws, outs = cache8.Workspace.for_cache(cache, heads, rows), []
    for _ in range(100):
        outs.append(torch.zeros_like(q))
        cache8.attention(cache, q, outs[-1], start, num_heads=heads, row_start=row_start, max_rows=rows, workspace=ws)
    assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_captured_step_serves_every_position():
    b = Batch(2, 256, 8, 2, 128)
    b.append([0, 0], [126, 60])
    qkv = torch.zeros((2, b.width), dtype=torch.float16, device="cuda")
    q, out, start = torch.zeros((2, 1024), dtype=torch.float16, device="cuda"), torch.zeros((2, 1024), dtype=torch.float16, device="cuda"), ints([126, 60])
    ws = cache8.Workspace.for_cache(b.cache, 8)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        cache8.append(b.cache, qkv, q, start, num_heads=8, bias=b.bias, rope=b.rope, flags=_lib.TWM_FLAG_PDL)
        cache8.attention(b.cache, q, out, start, num_heads=8, workspace=ws, flags=_lib.TWM_FLAG_PDL)
    for i in range(8):
        qkv.copy_(b.make(2))
        start.copy_(ints([126 + i, 60 + i]))
        graph.replay()
        for s, at in enumerate((126 + i, 60 + i)):
            qs, k, v = ref.project(qkv[s:s + 1], torch.tensor([at], device="cuda"), 8, 2, 128, b.bias, b.rope)
            b.held.append(s, at, k, v)
            want, off = ref.attention(qs, *b.held.held(s, at + 1), at, 8, 1 / math.sqrt(128), 0)
            assert bool(((out[s:s + 1].double() - want).abs() <= off).all())
    b.held.check(b.cache)


def test_other_stream_and_own_workspace():
    b = Batch(1, 4096, 16, 4, 128)
    b.append([0], [4000])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    q = 2 * torch.randn((1, 2048), generator=b.gen, device="cuda").half()
    out, here = torch.zeros_like(q), torch.zeros_like(q)
    torch.cuda.synchronize()
    cache8.attention(b.cache, q, out, ints([3999]), num_heads=16, stream=side)
    side.synchronize()
    cache8.attention(b.cache, q, here, ints([3999]), num_heads=16)
    assert torch.equal(out, here)


def test_rows_said_wrongly_stay_inside():
    """row_start that runs backwards, past the rows or below zero, and more rows than max_rows: nothing outside is touched."""
    b = Batch(3, 128, 4, 2, 64)
    b.append([0, 0, 0], [100, 100, 100])
    q = torch.randn((8, 256), generator=b.gen, device="cuda").half()
    for rows in ([-5, 2, 4, 9], [0, 6, 3, 8], [0, 100, 200, 300], [2, 2, 2, 2]):
        buf = torch.full((12, 256), 7.0, dtype=torch.float16, device="cuda")
        cache8.attention(b.cache, q, buf[:8], ints([50, -1, 90]), num_heads=4, row_start=ints(rows), max_rows=2)
        qkv = torch.randn((8, 512), generator=b.gen, device="cuda").half()
        cache8.append(b.cache, qkv, buf[:8], ints([100, -1, 90]), num_heads=4, row_start=ints(rows), max_rows=2)
        assert bool((buf[8:] == 7.0).all())


@pytest.mark.parametrize("heads,kv_heads,dim,rows", [(7, 1, 128, 1), (12, 1, 64, 1), (4, 1, 64, 3), (4, 1, 128, 30)])
def test_many_sequences(heads, kv_heads, dim, rows):
    """More sequences than warps look at by themselves, some of them out of the call or without a row."""
    seqs = 300
    b = Batch(seqs, 192, heads, kv_heads, dim)
    lengths = [rows + 7 * s % (192 - rows + 1) for s in range(seqs)]
    b.append([0] * seqs, lengths)
    counts = [0 if s % 11 == 5 else 1 + s % rows for s in range(seqs)]
    b.attend([-1 if s % 13 == 3 else n - c for s, (n, c) in enumerate(zip(lengths, counts))], counts, pad=1)


@pytest.mark.parametrize("rows", [1, 3, 70])
def test_up_to_the_capacity(rows):
    """The last places of a full cache, rows of which some or all lie behind them, and a sequence that stands past the end."""
    b = Batch(3, 256, 8, 2, 128)
    b.append([0, 0, 0], [256, 256, 256])
    b.attend([256 - rows] * 3, [rows] * 3)
    q = 2 * torch.randn((3 * rows, 1024), generator=b.gen, device="cuda").half()
    out = torch.full_like(q, 7.0)
    starts, row_start = [256 - rows // 2, 256, 1 << 30], ints([0, rows, 2 * rows, 3 * rows])
    cache8.attention(b.cache, q, out, ints(starts), num_heads=8, row_start=row_start, max_rows=rows)
    assert bool((out[rows // 2:] == 7.0).all())
    if rows > 1:
        want, off = ref.attention(q[:rows // 2], *b.held.held(0, 256), starts[0], 8, 1 / math.sqrt(128), 0)
        assert bool(((out[:rows // 2].double() - want).abs() <= off).all())
    before = [t.clone() for t in (b.cache.k.view(torch.uint8), b.cache.v.view(torch.uint8), b.cache.k_tail, b.cache.v_tail)]
    qkv = torch.randn((3 * rows, b.width), generator=b.gen, device="cuda").half()
    cache8.append(b.cache, qkv, out, ints([256, 256, 1 << 30]), num_heads=8, row_start=row_start, max_rows=rows)
    assert all(torch.equal(x, t) for x, t in zip(before, (b.cache.k.view(torch.uint8), b.cache.v.view(torch.uint8), b.cache.k_tail, b.cache.v_tail)))


@pytest.mark.parametrize("rows", [1, 2, 9])
def test_more_query_heads_than_rows_of_a_tile(rows):
    b = Batch(2, 320, 300, 1, 64)
    b.append([0, 0], [200, 31])
    b.attend([200 - rows, 31 - rows], [rows, rows])
    b.attend([200 - rows, 31 - rows], [rows, rows], window=(1 << 31) - 1)


def test_two_captured_calls_at_once():
    """Two graphs with workspaces of their own, of few rows and of many, run on two streams together."""
    b = Batch(4, 2048, 16, 4, 128)
    b.append([0] * 4, [2000, 1500, 1999, 700])
    calls = []
    for rows in (1, 64):
        start, row_start = ints([2000 - rows, 1500 - rows, 1999 - rows, 700 - rows]), ints([rows * s for s in range(5)])
        q = 2 * torch.randn((4 * rows, 2048), generator=b.gen, device="cuda").half()
        for _ in range(2):
            out, ws = torch.zeros_like(q), cache8.Workspace.for_cache(b.cache, 16, rows)
            graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.graph(graph, stream=side):
                for _ in range(3):
                    cache8.attention(b.cache, q, out, start, num_heads=16, row_start=row_start, max_rows=rows, workspace=ws, flags=_lib.TWM_FLAG_PDL)
            want = torch.zeros_like(q)
            cache8.attention(b.cache, q, want, start, num_heads=16, row_start=row_start, max_rows=rows)
            calls.append((graph, side, out, want, (start, row_start, q, ws)))      # a graph does not keep what it uses
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, side, *_ in calls:
            with torch.cuda.stream(side):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, _, out, want, _ in calls)


@pytest.mark.parametrize("rows", [1, 30])
def test_append_in_place(rows):
    """The rotated queries over those of the fused projection."""
    b = Batch(2, 128, 8, 2, 128)
    qkv = b.make(2 * rows).half()
    want, place, row_start = torch.zeros((2 * rows, 1024), dtype=torch.float16, device="cuda"), qkv.clone(), ints([0, rows, 2 * rows])
    kw = dict(num_heads=8, row_start=row_start, max_rows=rows, bias=b.bias, rope=b.rope)
    cache8.append(b.cache, qkv, want, ints([0, 0]), **kw)
    cache8.append(b.cache, place, place[:, :1024], ints([0, 0]), **kw)
    assert torch.equal(place[:, :1024], want) and torch.equal(place[:, 1024:], qkv[:, 1024:])


def test_calls_without_rows():
    b = Batch(2, 128, 8, 2, 64)
    b.append([0, 0], [70, 3])
    none = torch.zeros((0, b.width), dtype=torch.float16, device="cuda")
    cache8.append(b.cache, none, none[:, :512], ints([70, 3]), num_heads=8, row_start=ints([0, 0, 0]))
    cache8.attention(b.cache, none[:, :512], none[:, :512], ints([70, 3]), num_heads=8, row_start=ints([0, 0, 0]))
    b.held.check(b.cache)
    with pytest.raises(_lib.TwmError):
        cache8.attention(b.cache, none[:, :512], none[:, :512], ints([70, 3]), num_heads=8)


def verify_copies(b, length, rows, window, scale, copies):
    """Attention over as many copies of the batch's one sequence, so that a CTA has a run of many units; what the runs begin and end with differs."""
    c = b.cache
    many = lambda t: t.view(torch.uint8 if t.dtype.itemsize == 1 else t.dtype).expand(copies, *t.shape[1:]).contiguous()  # noqa: E731
    cache = cache8.Cache8(*(many(t) for t in (c.k, c.v, c.k_scale, c.v_scale, c.k_tail, c.v_tail)))
    one = torch.rand((rows, b.heads * b.dim), generator=b.gen, device="cuda").half() + 0.5
    q = one.repeat(copies, 1)
    out = torch.zeros_like(q)
    cache8.attention(cache, q, out, ints([length - rows] * copies), num_heads=b.heads, row_start=ints([rows * s for s in range(copies + 1)]), max_rows=rows,
                     window=window, scale=scale)
    want, off = ref.attention_by_values(one, *b.held.held(0, length), length - rows, b.heads, scale, window)
    worst = ((out.double().unflatten(0, (copies, rows)) - want).abs() / off).max()
    assert bool(worst <= 1), (length, window, float(worst))


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 1, 128), (2, 2, 64)])
@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("size", [1e-4, 1e-3, 1e-2, 1.0])
@pytest.mark.parametrize("blocks", ["alike", "zeros first", "zeros between", "zeros in the tail", "units of one", "larger tail", "smaller tail", "zeros"])
def test_small_values_keep_their_bits(heads, kv_heads, dim, rows, size, blocks):
    """Values of any size, beside blocks or a tail of zeros, of values whose scale is one, and of larger and smaller ones."""
    def make(n):
        x = torch.randn((n, (heads + 2 * kv_heads) * dim), generator=gen("v", n, dim), device="cuda")
        block = torch.arange(n, device="cuda")[:, None] // 64
        tail = block == n // 64
        v = x[:, (heads + kv_heads) * dim:]
        v *= size
        if blocks.startswith("zeros"):
            v *= ~{"zeros": block >= 0, "zeros first": block == 0, "zeros between": (block == 2) | (block == 5), "zeros in the tail": tail}[blocks]
        elif blocks == "units of one":
            v *= torch.where(block == 6, 60.0 / size, 1.0)
        elif blocks != "alike":
            v *= torch.where(tail, 2.0 ** 5 if blocks == "larger tail" else 2.0 ** -5, 1.0)
        return x
    for length in (448, 451, 500):
        b = Batch(1, 512, heads, kv_heads, dim, bias=False, rope=False, make=make)
        b.append([0], [length])
        for window in (0, 8, 70):
            verify_copies(b, length, rows, window, 1 / math.sqrt(dim), 400 if rows < 9 else 40)


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 1, 128), (2, 2, 64)])
@pytest.mark.parametrize("rows", [1, 3, 40, 70])
@pytest.mark.parametrize("size", [1e-4, 1e-3, 1e-2])
@pytest.mark.parametrize("where", ["tail", "zeros", "zeros of one warp"])
def test_equal_weights_of_small_values(heads, kv_heads, dim, rows, size, where):
    """All tokens but those of the tail, or of a block of zeros, weigh the same, so that what a weight is off by does not average out."""
    length = 64 * 7 + (40 if where == "tail" else 0)

    def make(n):
        x = torch.zeros((n, heads + 2 * kv_heads, dim), device="cuda")
        token = torch.arange(n, device="cuda")[:, None]
        other = token // 64 == (7 if where == "tail" else 1)
        x[:, heads:heads + kv_heads, 0] = torch.where(other, 0.25, 0.0)
        v = size * (1 + torch.rand((n, kv_heads, dim), generator=gen("w", n), device="cuda"))
        none = {"tail": other & False, "zeros": other, "zeros of one warp": other & (token % 64 < 16)}[where]
        x[:, heads + kv_heads:] = torch.where(none[:, :, None], 0.0, v)
        return x.flatten(1)
    b = Batch(1, 512, heads, kv_heads, dim, bias=False, rope=False, make=make)
    b.append([0], [length])
    for window in (0, 300):
        verify_copies(b, length, rows, window, 1.0, 400 if rows < 9 else 40)


@pytest.mark.parametrize("rows,most", [(1, 2), (3, 40), (20, 64)])
def test_room_for_more_rows_than_the_call_has(rows, most):
    """max_rows, and a workspace for as many, above the call's rows: what a program keeps for its largest calls serves the small ones."""
    b = Batch(1, 256, 8, 2, 128)
    b.append([0], [130])
    ws = cache8.Workspace.for_cache(b.cache, 8, most)
    qkv = b.make(rows).half()
    q, out = torch.zeros((rows, 1024), dtype=torch.float16, device="cuda"), torch.zeros((rows, 1024), dtype=torch.float16, device="cuda")
    kw = dict(num_heads=8, row_start=ints([0, rows]), max_rows=most)
    cache8.append(b.cache, qkv, q, ints([130]), bias=b.bias, rope=b.rope, **kw)
    qs, k, v = ref.project(qkv, torch.arange(130, 130 + rows, device="cuda"), 8, 2, 128, b.bias, b.rope)
    b.held.append(0, 130, k, v)
    b.held.check(b.cache)
    cache8.attention(b.cache, q, out, ints([130]), workspace=ws, **kw)
    want, off = ref.attention(qs, *b.held.held(0, 130 + rows), 130, 8, 1 / math.sqrt(128), 0)
    assert torch.equal(q, qs) and bool(((out.double() - want).abs() <= off).all())


def test_single_rows_of_any_stride():
    """One row has no next one: a transposed column, and a row of a buffer whose width is odd."""
    b = Batch(1, 128, 8, 2, 128)
    b.append([0], [70])
    columns = b.make(1).half()[0]
    qs, k, v = ref.project(columns[None], torch.tensor([70], device="cuda"), 8, 2, 128, b.bias, b.rope)
    b.held.append(0, 70, k, v)
    want, off = ref.attention(qs, *b.held.held(0, 71), 70, 8, 1 / math.sqrt(128), 0)
    for place in (lambda n: torch.zeros((n, 1), dtype=torch.float16, device="cuda").t(), lambda n: torch.zeros((1, n + 3), dtype=torch.float16, device="cuda")[:, :n]):
        qkv, q, out = place(b.width), place(1024), place(1024)
        qkv.copy_(columns[None])
        assert qkv.stride(0) not in (b.width,) and qkv.stride(1) == 1
        cache8.append(b.cache, qkv, q, ints([70]), num_heads=8, bias=b.bias, rope=b.rope)
        b.held.check(b.cache)
        cache8.attention(b.cache, q, out, ints([70]), num_heads=8)
        assert torch.equal(q, qs) and bool(((out.double() - want).abs() <= off).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("first", ["zeros", "units of one"])
def test_second_half_behind_a_tile_without_it(dim, first):
    """280 rows a sequence, a tile of 256 and one of 24: the rows of the second half come to the next sequence's first block, whose scale is one, ahead
    of its values."""
    def make(n):
        x = torch.zeros((n, 6, dim), device="cuda")
        token = torch.arange(n, device="cuda")[:, None]
        x[:, 4:5, 0] = torch.where(token < 64, 0.25, 0.0)
        v = 1e-4 * (1 + torch.rand((n, 1, dim), generator=gen("half", n), device="cuda"))
        x[:, 5:] = torch.where((token < 64)[:, :, None], 0.0 if first == "zeros" else 230.0, v)
        return x.flatten(1)
    b = Batch(1, 512, 4, 1, dim, bias=False, rope=False, make=make)
    b.append([0], [448])
    for _ in range(3):
        verify_copies(b, 448, 70, 0, 1.0, 300)
