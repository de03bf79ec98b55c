"""GPU tests of sampling against its definition in 64 bits."""
import math
import zlib

import numpy as np
import pytest
import torch

from tensorwarp_b200 import _lib, sampling

pytestmark = pytest.mark.gpu


def gen(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def chosen(row, u, t, top_k=0, top_p=1.0, min_p=0.0):
    """(token, its share, exponents of the token and of the average kept one) by the definition; row: f64."""
    row = np.where(np.isnan(row), -np.inf, row)
    if not t > 0 or row.max() == -np.inf:
        return int(row.argmax()), 1.0, 0.0
    order = np.lexsort((np.arange(row.size), -row))
    if top_k > 0:
        order = order[:top_k]
    top = row[order[0]]
    with np.errstate(invalid="ignore"):
        x = (row - top) / t
    x[row == top] = 0.0
    w = np.where(row == -np.inf, 0.0, np.exp(x))
    if top_p < 1:
        before = np.concatenate(([0.0], np.cumsum(w[order])[:-1]))
        order = order[:max(1, int((before < top_p * w[order].sum()).sum()))]
    order = np.sort(order[w[order] >= min(min_p, 1.0)])
    run = np.cumsum(w[order])
    at = min(int(np.searchsorted(run, u * run[-1], side="right")), order.size - 1)
    while w[order[at]] == 0:
        at -= 1
    live = w[order] > 0
    size = -x[order[at]] + float((w[order][live] * -x[order][live]).sum() / run[-1])
    return int(order[at]), float(w[order[at]] / run[-1]), size


# How far a border may lie from where it should: weights are FP32 exponentials, off by a few 2^-24 each and by as much for every unit of their
# exponent, so running sums are off by less than 2^-19 of the whole.
NEAR = 2.0 ** -19


def verify(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, **kw):
    rows = logits.shape[0]
    tokens = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    prob = torch.full((rows,), -7.0, device="cuda")
    sampling.sample(logits, u, tokens, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, prob=prob, **kw)
    torch.cuda.synchronize()
    host = logits.double().cpu().numpy()
    pick = lambda t, r, default: default if t is None else t[r].item()  # noqa: E731
    for r in range(rows):
        t, k, p, m, x = pick(temperature, r, 1.0), pick(top_k, r, 0), pick(top_p, r, 1.0), pick(min_p, r, 0.0), float(u[r])
        want = [chosen(host[r], x, t, k, p, m)]
        if int(tokens[r]) != want[0][0]:           # next to a border either side will do
            want += [chosen(host[r], min(max(x + a, 0.0), 1.0), t, k, q, n) for a in (-NEAR, 0, NEAR)
                     for q in ((p,) if p >= 1 else (p - NEAR, p, min(p + NEAR, 1.0))) for n in ((m,) if m <= 0 else (m * (1 - NEAR), m, m * (1 + NEAR)))]
        same = [w for w in want if w[0] == int(tokens[r])]
        assert same, (r, int(tokens[r]), want[0], t, k, p, m, x)
        # w and the sum of w: 4 roundings of the exponent and 8 of the numbers themselves
        assert any(abs(float(prob[r]) - w[1]) <= w[1] * (4 * w[2] + 16) * 2.0 ** -24 for w in same), (r, float(prob[r]), same[0])
    return tokens


def f32(values):
    return torch.tensor(values, dtype=torch.float32, device="cuda")


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=5), dict(top_k=50, top_p=0.9), dict(top_p=0.5), dict(top_p=0.95, temperature=1.5), dict(min_p=0.1),
            dict(top_k=700, top_p=0.99, min_p=0.001, temperature=2.0), dict(temperature=0.05), dict(temperature=0.0), dict(top_p=0.999, temperature=5.0),
            dict(top_k=20, min_p=0.02), dict(top_p=1e-6), dict(min_p=1.0), dict(temperature=100.0, top_p=0.7)]


@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 1025, 32768, 32771, 152064, 262144])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("spread", [0.1, 3.0, 30.0])
def test_settings(vocab, dtype, spread):
    g = gen(vocab, spread)
    rows = len(SETTINGS)
    logits = (spread * torch.randn((rows, vocab), generator=g, device="cuda")).to(dtype)
    u = torch.rand(rows, generator=g, device="cuda")
    verify(logits, u, f32([s.get("temperature", 1.0) for s in SETTINGS]), i32([s.get("top_k", 0) for s in SETTINGS]),
           f32([s.get("top_p", 1.0) for s in SETTINGS]), f32([s.get("min_p", 0.0) for s in SETTINGS]))


@pytest.mark.parametrize("rows", [1, 3, 37, 200, 1000])
def test_rows(rows):
    g = gen("rows", rows)
    logits = 2.5 * torch.randn((rows, 5003), generator=g, device="cuda")
    u = torch.rand(rows, generator=g, device="cuda")
    pick = [SETTINGS[r % len(SETTINGS)] for r in range(rows)]
    a = verify(logits, u, f32([s.get("temperature", 1.0) for s in pick]), i32([s.get("top_k", 0) for s in pick]),
               f32([s.get("top_p", 1.0) for s in pick]), f32([s.get("min_p", 0.0) for s in pick]))
    b = verify(logits, u, f32([s.get("temperature", 1.0) for s in pick]), i32([s.get("top_k", 0) for s in pick]),
               f32([s.get("top_p", 1.0) for s in pick]), f32([s.get("min_p", 0.0) for s in pick]))
    assert torch.equal(a, b)


@pytest.mark.parametrize("vocab", [3, 64, 5000, 152064])
@pytest.mark.parametrize("setting", [dict(), dict(top_k=3), dict(top_p=0.4), dict(top_k=40, top_p=0.5), dict(min_p=1.0), dict(temperature=0.0), dict(top_k=2000)])
def test_equal_numbers(vocab, setting):
    """A row of one number, of two, of both zeros: ties go to the lowest index."""
    logits = torch.zeros((4, vocab), device="cuda")
    logits[1] = -3.5
    logits[2, vocab // 2:] = 1.0
    logits[3, ::2] = -0.0
    for u in (0.0, 0.3, 0.99):
        one = lambda k, make, other: None if k not in setting else make([setting[k]] * 4)  # noqa: E731
        verify(logits, f32([u] * 4), one("temperature", f32, 1.0), one("top_k", i32, 0), one("top_p", f32, 1.0), one("min_p", f32, 0.0))


def test_numbers_that_are_none():
    """-inf and NaN never win; +inf shares with other +inf only; a row without a number gives token 0."""
    inf, nan = math.inf, math.nan
    n = 2000
    logits = torch.full((8, n), -inf, device="cuda")
    logits[0, 5] = -1e30
    logits[1] = nan
    logits[2, 7], logits[2, 1500], logits[2, 30] = inf, inf, 3.4e38
    logits[3, ::3] = nan
    logits[3, 1::3] = torch.randn(667, generator=gen("n"), device="cuda")
    logits[5, 1999] = 3.4e38
    logits[5, 0] = -3.4e38
    logits[6] = nan
    logits[6, 1234] = 1.0
    logits[7, :2] = 3.4e38
    for u in (0.0, 0.4, 0.9999):
        for setting in (dict(), dict(top_k=i32([2] * 8)), dict(top_p=f32([0.6] * 8)), dict(min_p=f32([0.5] * 8)), dict(temperature=f32([0.0] * 8)),
                        dict(top_k=i32([1999] * 8), top_p=f32([0.99] * 8))):
            got = verify(logits, f32([u] * 8), **setting)
            assert got[0] == 5 and got[1] == 0 and int(got[2]) in (7, 1500) and got[4] == 0 and got[5] == 1999 and got[6] == 1234 and int(got[7]) in (0, 1)


def test_ends_of_the_random_numbers():
    logits = torch.randn((6, 3000), generator=gen("e"), device="cuda")
    logits[:, :10], logits[:, -10:] = -math.inf, -math.inf
    u = f32([0.0, 1.0, -1.0, 2.0, math.nan, 1 - 2.0 ** -24])
    tokens = torch.zeros(6, dtype=torch.int32, device="cuda")
    sampling.sample(logits, u, tokens)
    assert tokens.tolist()[0] == 10 and tokens.tolist()[2] == 10 and tokens.tolist()[4] == 10
    assert tokens.tolist()[1] == 2989 and tokens.tolist()[3] == 2989


def test_settings_past_their_ranges():
    """A cut below its range keeps the first token, one past it keeps all."""
    logits = torch.randn((1, 3000), generator=gen("r"), device="cuda")
    first = int(logits[0].argmax())
    for setting, alike in ((dict(top_p=0.0), None), (dict(top_p=-1.0), None), (dict(min_p=2.0), None), (dict(top_p=5.0), {}), (dict(min_p=-3.0), {}), (dict(top_k=-4), {}),
                           (dict(top_k=3000), {}), (dict(top_k=1 << 30), {}), (dict(temperature=-1.0), None), (dict(temperature=math.nan), None)):
        args = {k: (i32 if k == "top_k" else f32)([v]) for k, v in setting.items()}
        for u in (0.1, 0.77):
            tokens, plain = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
            sampling.sample(logits, f32([u]), tokens, **args)
            sampling.sample(logits, f32([u]), plain)
            assert int(tokens) == (first if alike is None else int(plain)), setting


def test_row_strides_and_odd_places():
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        wide = (3 * torch.randn((5, 40009), generator=gen("w"), device="cuda")).to(dtype)
        u = torch.rand(5, generator=gen("v"), device="cuda")
        for a, b in ((0, 40000), (1, 40000), (3, 39998), (8, 33000)):
            verify(wide[:, a:b], u, top_k=i32([50] * 5), top_p=f32([0.9] * 5))


def test_frequencies():
    """Shares of the tokens over evenly spread random numbers are those of the distribution, to one random number each border."""
    n, rows = 12, 4096
    logits = torch.randn((1, n), generator=gen("f"), device="cuda").expand(rows, n)
    u = (torch.arange(rows, device="cuda") + 0.5) / rows
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    sampling.sample(logits.contiguous(), u, tokens, top_k=i32([7] * rows))
    w = torch.softmax(logits[0].double(), 0)
    kept = torch.topk(w, 7).indices
    share = torch.zeros_like(w)
    share[kept] = w[kept] / w[kept].sum()
    count = torch.bincount(tokens.long(), minlength=n).double()
    assert bool(((count - share * rows).abs() <= 1.001).all()) and bool((tokens[1:] >= tokens[:-1]).all())


def test_decode_loop_form():
    """Random numbers by the step counter, history, and the counters advanced; a full list is not written past its end."""
    n, steps = 5000, 5
    logits = 2 * torch.randn((1, n), generator=gen("d"), device="cuda")
    u = torch.rand(3, generator=gen("c"), device="cuda")
    tokens, step, pos, length = (torch.full((1,), v, dtype=torch.int32, device="cuda") for v in (0, 0, 40, 41))
    history = torch.full((4,), -1, dtype=torch.int32, device="cuda")
    args = _lib.SampleArgs(1, n, _lib.TWM_F32, logits.data_ptr(), n, u.data_ptr(), None, None, None, None, tokens.data_ptr(), None, step.data_ptr(), 3,
                           history.data_ptr(), 3, pos.data_ptr(), length.data_ptr())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _lib.check(_lib.lib().twm_sample(_lib.C.addressof(args), _lib.TWM_FLAG_PDL, torch.cuda.current_stream().cuda_stream), "twm_sample")
    want = [chosen(logits[0].double().cpu().numpy(), float(u[min(i, 2)]), 1.0)[0] for i in range(steps)]
    for i in range(steps):
        graph.replay()
        assert int(tokens) == want[i]
    assert history.tolist() == want[:3] + [-1] and int(step) == steps and int(pos) == 40 + steps and int(length) == 41 + steps


def test_other_stream():
    logits = torch.randn((9, 30000), generator=gen("o"), device="cuda")
    u = torch.rand(9, generator=gen("p"), device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    tokens, here = torch.zeros(9, dtype=torch.int32, device="cuda"), torch.zeros(9, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    sampling.sample(logits, u, tokens, top_p=f32([0.9] * 9), stream=side)
    side.synchronize()
    sampling.sample(logits, u, here, top_p=f32([0.9] * 9))
    assert torch.equal(tokens, here)


@pytest.mark.parametrize("vocab", [655361, 700001, 1 << 20])
def test_largest_vocabularies(vocab):
    """Rows of which a CTA's slice does not fit its shared memory."""
    g = gen("largest", vocab)
    pick = [SETTINGS[i] for i in (0, 4, 5, 8, 10, 13, 15)]
    logits = 3.0 * torch.randn((len(pick), vocab), generator=g, device="cuda")
    verify(logits, torch.rand(len(pick), generator=g, device="cuda"), f32([s.get("temperature", 1.0) for s in pick]), i32([s.get("top_k", 0) for s in pick]),
           f32([s.get("top_p", 1.0) for s in pick]), f32([s.get("min_p", 0.0) for s in pick]))


def test_two_calls_at_once():
    g = gen("two")
    logits = [3.0 * torch.randn((150, 50000), generator=g, device="cuda") for _ in range(2)]
    u, p = torch.rand(150, generator=g, device="cuda"), f32([0.9] * 150)
    want = [torch.zeros(150, dtype=torch.int32, device="cuda") for _ in range(2)]
    got = [torch.zeros(150, dtype=torch.int32, device="cuda") for _ in range(2)]
    for x, t in zip(logits, want):
        sampling.sample(x, u, t, top_p=p)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for x, t, s in zip(logits, got, streams):
            sampling.sample(x, u, t, top_p=p, stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, got))


@pytest.mark.parametrize("vocab", [700, 32771, 152064])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_equal_numbers_at_the_border_of_top_k(vocab, dtype):
    """A few dozen different logits, so that hundreds are equal where top-k ends, and top-p behind it: a hundred calls, one result."""
    g = gen("border", vocab)
    ks, ps = [60, 100, 333, 600], [0.2, 0.5, 0.9, 0.999]
    rows = len(ks) * len(ps)
    logits = (torch.randint(0, 12, (rows, vocab), generator=g, device="cuda") * 0.25).to(dtype)
    u = torch.rand(rows, generator=g, device="cuda")
    top_k, top_p = i32([k for k in ks for _ in ps]), f32([p for _ in ks for p in ps])
    want = verify(logits, u, top_k=top_k, top_p=top_p)
    got = [torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(100)]
    for t in got:
        sampling.sample(logits, u, t, top_k=top_k, top_p=top_p)
    assert all(torch.equal(t, want) for t in got)


@pytest.mark.parametrize("vocab", [5, 3000, 152064])
def test_infinite_temperature(vocab):
    """All finite logits weigh the same, whatever cut is asked for, and the loop's counters advance."""
    cuts = [dict(), dict(min_p=1.0), dict(min_p=0.5), dict(min_p=3.0), dict(top_k=3), dict(top_k=1000, min_p=1.0), dict(top_p=0.3), dict(top_p=0.9, min_p=1.0),
            dict(top_k=200, top_p=0.5, min_p=0.1)]
    logits = 5 * torch.randn((len(cuts), vocab), generator=gen("inf", vocab), device="cuda")
    logits[:, 1], logits[:, 3] = -math.inf, math.nan
    for u in (0.0, 0.37, 0.999):
        verify(logits, f32([u] * len(cuts)), f32([math.inf] * len(cuts)), i32([c.get("top_k", 0) for c in cuts]), f32([c.get("top_p", 1.0) for c in cuts]),
               f32([c.get("min_p", 0.0) for c in cuts]))
    tokens, step, pos, length = (torch.full((1,), v, dtype=torch.int32, device="cuda") for v in (-1, 0, 7, 8))
    u, t, m = f32([0.5]), f32([math.inf]), f32([1.0])
    args = _lib.SampleArgs(1, vocab, _lib.TWM_F32, logits.data_ptr(), vocab, u.data_ptr(), t.data_ptr(), None, None, m.data_ptr(), tokens.data_ptr(), None, step.data_ptr(),
                           1, None, 0, pos.data_ptr(), length.data_ptr())
    _lib.check(_lib.lib().twm_sample(_lib.C.addressof(args), 0, torch.cuda.current_stream().cuda_stream), "twm_sample")
    assert int(tokens) >= 0 and int(step) == 1 and int(pos) == 8 and int(length) == 9


@pytest.mark.parametrize("vocab", [50, 3000, 18169, 152064])
def test_tokens_without_weight_do_not_move_a_border(vocab):
    """Two equal logits far above all others: at a half of the mass top-p keeps the first one, whatever top-k leaves beside them."""
    ks = [0, 2, vocab // 2, vocab - 1, vocab]
    logits = torch.round(torch.randn((len(ks), vocab), generator=gen("weight", vocab), device="cuda").clamp(-2, 2))
    first, second = vocab // 3, vocab - 2
    logits[:, first] = logits[:, second] = 4.0
    for u in (0.1, 0.9):
        for p, want, share in ((0.5, first, 1.0), (0.75, first if u < 0.5 else second, 0.5)):
            tokens, prob = torch.zeros(len(ks), dtype=torch.int32, device="cuda"), torch.zeros(len(ks), device="cuda")
            sampling.sample(logits, f32([u] * len(ks)), tokens, temperature=f32([1e-4] * len(ks)), top_k=i32(ks), top_p=f32([p] * len(ks)), prob=prob)
            assert tokens.tolist() == [want] * len(ks) and prob.tolist() == [share] * len(ks), (u, p)
