"""CPU tests of what the cache held in 8 bits and sampling refuse; nothing here makes a CUDA call."""
import ctypes as C

import pytest
import torch

from tensorwarp_b200 import _lib, cache8, sampling
from tensorwarp_b200.scheduler import Scheduler


def cache(**kw):
    fields = dict(seqs=2, kv_heads=4, head_dim=128, capacity=256, k=0x10000, v=0x20000, k_scale=0x30000, v_scale=0x40000, k_tail=0x50000, v_tail=0x60000)
    fields.update(kw)
    return _lib.Cache8(**fields)


def append(lib, c, q=0x1000, ldq=1024, qkv=0x2000, ldqkv=2048, bias=None, rope=None, heads=8, rows=2, row_start=None, max_rows=1, start=0x3000):
    args = _lib.Cache8AppendArgs(q, ldq, qkv, ldqkv, bias, rope, heads, rows, max_rows, row_start, start)
    return lib.twm_cache8_append(C.addressof(c) if c is not None else None, C.addressof(args), 0, None)


def attention(lib, c, out=0x1000, ldo=1024, q=0x2000, ldq=1024, heads=8, rows=2, row_start=None, max_rows=1, start=0x3000, scale=0.1, window=0, ws=0x4000,
              nbytes=1 << 40):
    args = _lib.Cache8AttentionArgs(out, ldo, q, ldq, heads, rows, max_rows, window, row_start, start, ws, nbytes, scale)
    return lib.twm_cache8_attention(C.addressof(c) if c is not None else None, C.addressof(args), 0, None)


BAD_CACHES = [dict(seqs=0), dict(seqs=65536), dict(kv_heads=0), dict(head_dim=96), dict(head_dim=0), dict(capacity=100), dict(capacity=0), dict(k=None), dict(v=None),
              dict(k_scale=None), dict(v_scale=None), dict(k_tail=None), dict(v_tail=None), dict(seqs=60000, capacity=1 << 20)]


@pytest.mark.parametrize("call", [append, attention])
def test_caches_that_are_refused(twm_lib, call):
    assert call(twm_lib, None) == _lib.TWM_EINVAL
    for bad in BAD_CACHES:
        assert call(twm_lib, cache(**bad)) == _lib.TWM_EINVAL, bad
    for bad in (dict(k=0x10008), dict(v=0x20004), dict(k_tail=0x50002), dict(v_tail=0x60008)):
        assert call(twm_lib, cache(**bad)) == _lib.TWM_EALIGN, bad


@pytest.mark.parametrize("call", [append, attention])
def test_rows_that_are_refused(twm_lib, call):
    for bad in (dict(heads=0), dict(heads=6), dict(rows=0), dict(rows=3), dict(max_rows=0), dict(max_rows=2), dict(start=None), dict(q=None), dict(ldq=1016),
                dict(row_start=0x5000, rows=4, max_rows=5)):
        assert call(twm_lib, cache(), **bad) == _lib.TWM_EINVAL, bad
    for bad in (dict(ldq=1025), dict(q=0x1008)):
        assert call(twm_lib, cache(), **bad) == _lib.TWM_EALIGN, bad


def test_other_refusals(twm_lib):
    for bad in (dict(qkv=None), dict(ldqkv=2040)):
        assert append(twm_lib, cache(), **bad) == _lib.TWM_EINVAL, bad
    for bad in (dict(qkv=0x2002), dict(ldqkv=2052), dict(bias=0x7004), dict(rope=0x7008)):
        assert append(twm_lib, cache(), **bad) == _lib.TWM_EALIGN, bad
    for bad in (dict(out=None), dict(ldo=1000), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(ws=None)):
        assert attention(twm_lib, cache(), **bad) == _lib.TWM_EINVAL, bad
    for bad in (dict(out=0x1001), dict(ldo=1028), dict(ws=0x4008)):
        assert attention(twm_lib, cache(), **bad) == _lib.TWM_EALIGN, bad
    assert attention(twm_lib, cache(), nbytes=8) == _lib.TWM_EWORKSPACE


def test_no_arguments(twm_lib):
    assert twm_lib.twm_cache8_append(C.addressof(cache()), None, 0, None) == _lib.TWM_EINVAL
    assert twm_lib.twm_cache8_attention(C.addressof(cache()), None, 0, None) == _lib.TWM_EINVAL


def test_workspace_sizes(twm_lib):
    size = lambda c, heads, rows: twm_lib.twm_cache8_attention_bytes(C.addressof(c), heads, rows)  # noqa: E731
    assert twm_lib.twm_cache8_attention_bytes(None, 8, 1) == 0 and size(cache(), 0, 1) == 0 and size(cache(), 8, 0) == 0 and size(cache(head_dim=80), 8, 1) == 0
    assert size(cache(), 8, 1) > 0


def sample_args(**kw):
    fields = dict(rows=1, vocab=100, dtype=_lib.TWM_F32, logits=0x1000, ld=100, random=0x2000, tokens=0x3000)
    fields.update(kw)
    return _lib.SampleArgs(**fields)


def test_sampling_that_is_refused(twm_lib):
    assert twm_lib.twm_sample(None, 0, None) == _lib.TWM_EINVAL
    loop = dict(step=0x4000, random_count=3, pos=0x5000, len=0x6000)
    for bad in (dict(rows=0), dict(vocab=0), dict(vocab=(1 << 20) + 1, ld=1 << 21), dict(dtype=3), dict(logits=None), dict(ld=99), dict(random=None), dict(tokens=None),
                dict(loop, rows=2), dict(loop, random_count=0), dict(loop, pos=None), dict(loop, len=None), dict(loop, history=0x7000, history_capacity=0)):
        assert twm_lib.twm_sample(C.addressof(sample_args(**bad)), 0, None) == _lib.TWM_EINVAL, bad
    assert twm_lib.twm_sample(C.addressof(sample_args(logits=0x1002)), 0, None) == _lib.TWM_EALIGN


def test_host_tensors_are_refused():
    with pytest.raises(_lib.TwmError):
        sampling.sample(torch.zeros(1, 8), torch.zeros(1), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(_lib.TwmError):
        cache8.Cache8.empty(1, 64, 1, 64, device="cpu")


def test_sampling_params():
    sampling.SamplingParams(temperature=0.0, top_k=3, top_p=0.5, min_p=0.1)
    for bad in (dict(temperature=-1.0), dict(temperature=float("inf")), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.5),
                dict(min_p=-0.1), dict(min_p=1.1)):
        with pytest.raises(ValueError):
            sampling.SamplingParams(**bad)


class Drawing:
    """An engine whose tokens are its sequence's random numbers."""
    vocab, capacity, max_live = 1000, 64, 2

    def __init__(self):
        self.calls, self.live = [], {}

    def open(self):
        seq = min(set(range(self.max_live)) - set(self.live))
        self.live[seq] = 0
        return seq

    def close(self, seq):
        del self.live[seq]

    def step(self, seq, tokens, want=()):
        self.live[seq] += len(tokens)

    def greedy(self, seq, tokens, count):
        self.calls.append(("greedy", count))
        self.live[seq] += len(tokens) + count - 1
        return [7] * count

    def sample(self, seq, tokens, count, params, generator):
        self.calls.append(("sample", count, params))
        self.live[seq] += len(tokens) + count - 1
        return (torch.rand(count, generator=generator) * self.vocab).int().tolist()


def test_scheduler_hands_sampling_on():
    """Settings and generator go with the request: other bursts, the same tokens; a request without settings is greedy."""
    params, seen = sampling.SamplingParams(temperature=0.5, seed=5), []
    for burst in (1, 4, 16):
        sch = Scheduler(Drawing(), portion=4, burst=burst)
        requests = [sch.submit([1, 2, 3, 4, 5, 6], 10, sampling=params), sch.submit([9], 4), sch.submit([1], 10, sampling=params)]
        assert len(list(sch.run())) == 3
        assert {c[0] for c in sch.engine.calls} == {"greedy", "sample"} and all(c[2] is params for c in sch.engine.calls if c[0] == "sample")
        seen.append([r.generated for r in requests])
        assert requests[1].generated == [7] * 4 and requests[0].generated == requests[2].generated
    assert seen[0] == seen[1] == seen[2]


def test_scheduler_refuses_sampling_on_engines_without_it():
    class Greedy(Drawing):
        sample = property(lambda self: (_ for _ in ()).throw(AttributeError()))
    sch = Scheduler(Greedy())
    sch.submit([1], 2)
    with pytest.raises(ValueError):
        sch.submit([1], 2, sampling=sampling.SamplingParams())


def test_command_line_takes_settings():
    """Bad settings are refused before a model is loaded."""
    from tensorwarp_b200.__main__ import main
    with pytest.raises(ValueError):
        main(["generate", "--model", "/nowhere", "--tokens", "1", "--temperature", "-1"])
    with pytest.raises(SystemExit):
        main(["generate", "--model", "/nowhere", "--tokens", "1", "--kv-cache", "int4"])


def test_command_line_refuses_cuts_without_a_temperature():
    from tensorwarp_b200.__main__ import main
    with pytest.raises(SystemExit):
        main(["generate", "--model", "/nowhere", "--tokens", "1", "--top-p", "0.9"])


def test_refused_calls_draw_no_random_numbers():
    """A call that an engine refuses leaves the generator and the settings of its loop as they were."""
    from types import SimpleNamespace

    from tensorwarp_b200.engine import DenseEngine
    from tensorwarp_b200.models.tw_marlin import Q4StepEngine
    from tensorwarp_b200.state import StateError

    def touched(*a, **kw):
        raise AssertionError("a refused call has set the loop's numbers")

    dense = DenseEngine.__new__(DenseEngine)
    dense.vocab, dense.capacity, dense.stream, dense.state, dense._loop = 100, 20, None, SimpleNamespace(length=lambda seq: 10), SimpleNamespace(set=touched)
    q4 = Q4StepEngine(SimpleNamespace(cfg=SimpleNamespace(vocab=100, max_seq=20), generate_tw_marlin_graph=touched))
    q4._length = 10
    for engine in (dense, q4):
        generator, params = torch.Generator().manual_seed(3), sampling.SamplingParams()
        before = generator.get_state()
        for tokens, count in (([1, 2], 10), ([1], 1000), ([], 2), ([100], 2), ([-1, 4], 3)):
            with pytest.raises((ValueError, StateError)):
                engine.sample(0, tokens, count, params, generator)
            assert torch.equal(generator.get_state(), before), (type(engine).__name__, tokens, count)
        assert engine.sample(0, [1], 0, params, generator) == [] and torch.equal(generator.get_state(), before)


def test_rows_over_one_another_are_refused(twm_lib):
    """Results over what is still to be read: the same rows, shifted ones, and rows of other strides that meet somewhere; columns of one buffer do not."""
    base, ws = 0x1000000, 0x9000000
    def attend(out, ldo, q, ldq, rows=6):
        # a workspace that is too small: what is not refused for its rows is for that
        return attention(twm_lib, cache(seqs=rows), out=base + 2 * out, ldo=ldo, q=base + 2 * q, ldq=ldq, rows=rows, ws=ws, nbytes=8)
    for args in ((0, 1024, 0, 1024), (0, 1024, 1016, 1024), (8, 1024, 0, 1024), (0, 1024, 5 * 1024, 1024), (6 * 1024 - 8, 1024, 0, 1024), (0, 2048, 1016, 2048), (1032, 2048, 0, 2048),
                 (0, 2048, 1016 + 2048 * 3, 2048), (0, 2048, 1024, 3080), (4000, 1024, 0, 4096), (0, 1024, 0, 1024, 1), (0, 9000, 1016, 7000, 1)):
        assert attend(*args) == attend(args[2], args[3], args[0], args[1], *args[4:]) == _lib.TWM_EINVAL, args
    for args in ((0, 2048, 1024, 2048), (0, 2048, 1024 + 2048, 2048), (0, 1024, 6 * 1024, 1024), (0, 2048, 1024, 4096), (0, 1024, 1024, 1024, 1), (0, 4096, 1024, 8192),
                 (0, 2056, 1024, 2056)):
        assert attend(*args) == attend(args[2], args[3], args[0], args[1], *args[4:]) == _lib.TWM_EWORKSPACE, args
    # q_out among qkv's columns, of queries, keys and values: the queries' own or none
    append_at = lambda q, ldq, rows=6: append(twm_lib, cache(seqs=rows), q=base + 2 * q, ldq=ldq, qkv=base, ldqkv=3080, rows=rows)  # noqa: E731
    for args in ((8, 3080), (1024, 3080), (3080, 3080), (2040, 3080), (0, 1024), (0, 3088), (16, 1024, 1)):
        assert append_at(*args) == _lib.TWM_EINVAL, args


def test_a_larger_workspace_serves_fewer_rows(twm_lib):
    """What is enough for `max_rows` rows a sequence is enough for fewer."""
    for head_dim in (64, 128):
        for heads in (4, 8, 12, 20, 28, 64, 284):
            sizes = [twm_lib.twm_cache8_attention_bytes(C.addressof(cache(head_dim=head_dim)), heads, n) for n in range(1, 200)]
            assert sizes == sorted(sizes)


@pytest.mark.parametrize("architecture", ["Bidasun", "Zukotar"])
def test_the_8_bit_cache_is_refused_where_there_is_none(tmp_path, architecture):
    """The option's name is in the error, ahead of any weights; the 4-bit decoder's builder takes it."""
    import inspect

    from tensorwarp_b200 import registry
    from tensorwarp_b200.__main__ import main
    (tmp_path / "config.json").write_text('{"architecture": "%s"}' % architecture)
    for kind in ("e4m3", "f16"):
        with pytest.raises(ValueError, match="kv_cache is an option of the 4-bit decoder"):
            registry.load(str(tmp_path), kv_cache=kind)
        with pytest.raises(ValueError, match="kv_cache is an option of the 4-bit decoder"):
            main(["generate", "--model", str(tmp_path), "--tokens", "1", "--kv-cache", kind])
    assert "kv_cache" in inspect.signature(registry.builder_for({"architecture": "TWMarlinQ4"})).parameters
