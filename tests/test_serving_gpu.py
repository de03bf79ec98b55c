"""GPU tests of decode steps that end in the cache held in 8 bits and in sampling: the 4-bit decoder, the dense-weight decoders, requests."""
import json
import math

import numpy as np
import pytest
import torch

import bidasun_cases as cases
import cache8_ref as ref
from tensorwarp_b200 import _dense, _lib, cache8, dense, registry
from tensorwarp_b200.engine import DenseEngine
from tensorwarp_b200.generate import Q4Model, QuantizedGenerationEngine, TransformerConfig
from tensorwarp_b200.models import bidasun
from tensorwarp_b200.sampling import SamplingParams
from tensorwarp_b200.scheduler import Scheduler

pytestmark = pytest.mark.gpu
CFG = TransformerConfig(hidden=256, num_heads=6, num_kv_heads=2, head_dim=128, ffn=512, vocab=1000, layers=2, max_seq=300, group_size=128)
CONFIG = {"architecture": "TWMarlinQ4", "hidden": 256, "num_heads": 2, "num_kv_heads": 1, "head_dim": 128, "ffn": 512, "vocab": 512,
          "layers": 2, "max_seq": 200, "group_size": 128, "seed": 3}


@pytest.fixture(scope="module")
def model():
    m = Q4Model(CFG, seed=5)
    m.lm_head *= 8                                 # heads that tell tokens apart
    return m


def held(cache, length):
    """f64 keys and values of the cache's one sequence, from its tensors."""
    full, out = length // 64, []
    for codes, scale, tail in ((cache.k, cache.k_scale, cache.k_tail), (cache.v, cache.v_scale, cache.v_tail)):
        x = codes[0].double().unflatten(1, (-1, 64))[:, :full] * scale[0].double()[:, :full, None, None]
        out.append(torch.cat((x.flatten(1, 2), tail[0, :, full % 2, :length - 64 * full].double()), dim=1))
    return out


def test_decode_step_on_the_8_bit_cache(model):
    """Tokens over the borders of blocks: what the last layer's append and attention made of its projections, step by step."""
    eng = QuantizedGenerationEngine(model, kv_cache="e4m3")
    eng.prefill_random_kv(120)
    b, cache = eng.buf, eng.buf.cache8[-1]
    bias = model.layers[-1].bqkv
    eng.set_token(17)
    for at in range(120, 200):
        eng.step_eager()
        torch.cuda.synchronize()
        q, k, v = ref.project(b.qkv[None], torch.tensor([at], device="cuda"), CFG.num_heads, CFG.num_kv_heads, CFG.head_dim, bias, b.rope)
        assert torch.equal(b.query, q)
        tail = (cache.k_tail, cache.v_tail)
        for t, x in zip(tail, (k, v)):
            assert torch.equal(t[0, :, at // 64 % 2, at % 64], x[0])
        want, off = ref.attention(q, *held(cache, at + 1), at, CFG.num_heads, 1 / math.sqrt(CFG.head_dim), 0)
        assert bool(((b.attn.double() - want[0]).abs() <= off[0]).all()), at
    assert int(b.pos) == 200 and int(b.cache_len) == 201 and _lib.lib().twm_device_error(None, _lib.C.byref(_lib.C.c_uint())) == 0


def test_captured_steps_are_the_eager_ones(model):
    """The captured step on the 8-bit cache, greedy and sampled, gives what eager steps give; what the cache takes."""
    for sampling in (None, SamplingParams(temperature=0.9, top_k=50, top_p=0.95, min_p=0.01, seed=4)):
        outs = []
        for eager in (True, False):
            eng = QuantizedGenerationEngine(model, kv_cache="e4m3")
            eng.prefill_random_kv(50)
            if not eager:
                outs.append(eng.generate_tw_marlin_graph(3, 40, sampling))
                continue
            eng.set_token(3)
            if sampling is not None:
                eng.buf.loop.set(sampling, torch.rand(40, generator=sampling.generator()))
            torch.cuda.synchronize()
            with torch.cuda.stream(eng.stream):
                for _ in range(40):
                    eng.forward_decode_tw_marlin_graph(eng.stream.cuda_stream, sampling is not None)
            torch.cuda.synchronize()
            outs.append(eng.buf.history[:40].tolist())
        assert outs[0] == outs[1] and len(set(outs[0])) > 1
    # codes, a scale a block, and two blocks in FP16: 4096 tokens in 0.53 of the FP16 cache's bytes
    assert cache8.Cache8.empty(1, 4096, 2, 128).bytes() == 2 * 2 * (4096 * 128 + 4096 // 64 * 4 + 2 * 64 * 128 * 2) < 0.54 * (2 * 4096 * 2 * 128 * 2)


def choice(logits, u, p: SamplingParams):
    """The token of one row by the definition, f64; None next to a border."""
    x = logits.double().cpu().numpy()
    order = np.lexsort((np.arange(x.size), -x))[:p.top_k or x.size]
    w = np.exp((x[order] - x[order[0]]) / p.temperature)
    before = np.concatenate(([0.0], np.cumsum(w)[:-1]))
    near = np.abs(before - p.top_p * w.sum()).min() < 2e-6 * w.sum() if p.top_p < 1 else False
    order = order[:max(1, int((before < p.top_p * w.sum()).sum()))] if p.top_p < 1 else order
    order = np.sort(order[w[:order.size] >= p.min_p])
    run = np.cumsum(np.exp((x[order] - x.max()) / p.temperature))
    near |= np.abs(run - u * run[-1]).min() < 2e-6 * run[-1]
    return None if near else int(order[np.searchsorted(run, u * run[-1], side="right")])


@pytest.mark.parametrize("params", [SamplingParams(temperature=1.3, seed=1), SamplingParams(temperature=0.8, top_k=20, seed=2),
                                    SamplingParams(temperature=1.0, top_p=0.7, seed=3), SamplingParams(temperature=1.5, top_k=100, top_p=0.9, min_p=0.05, seed=4)])
def test_sampled_tokens_of_the_4_bit_decoder(model, params):
    """Every token drawn is the definition's, for the step's logits and the generator's next number."""
    eng = QuantizedGenerationEngine(model, kv_cache="e4m3")
    u = torch.rand(30, generator=params.generator())
    tokens = eng.generate_tw_marlin_graph(9, 30, params)
    again = QuantizedGenerationEngine(model, kv_cache="e4m3")
    again.set_position(0)
    again.set_token(9)
    for i, t in enumerate(tokens):
        again.set_token(9 if i == 0 else tokens[i - 1])
        again.step_eager()
        torch.cuda.synchronize()
        assert choice(again.buf.logits, float(u[i]), params) in (t, None), i


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sampled_tokens_of_a_dense_decoder(dtype):
    """A prompt, then drawn tokens: each is the definition's for the logits of a step by step run, and bursts do not matter."""
    cfg = cases.CASES["uneven"]
    spec, t = bidasun.parse_config(cfg), cases.weights(cfg, 7)
    make = lambda: DenseEngine(dense.DenseModel(spec, bidasun.model_tensors(spec, lambda n, s: t[n]), dtype), portion=16)  # noqa: E731
    prompt, params = [3, 50, 7, 99, 120] * 8, SamplingParams(temperature=1.4, top_k=60, top_p=0.95, min_p=0.001, seed=11)
    eng, plain = make(), make()
    seq, g = eng.open(), params.generator()
    tokens = eng.sample(seq, prompt, 5, params, g)
    tokens += eng.sample(seq, tokens[-1:], 1, params, g)
    tokens += eng.sample(seq, tokens[-1:], 19, params, g)
    u, other = torch.rand(25, generator=params.generator()), plain.open()
    logits = plain.step(other, prompt, [len(prompt) - 1])[0].clone()
    for i, token in enumerate(tokens):
        assert choice(logits, float(u[i]), params) in (token, None), i
        logits = plain.step(other, [token], [0])[0].clone()
    assert len(set(tokens)) > 5 and _dense.device_error() == 0
    assert eng.sample(seq, [1], 0, params, g) == []
    with pytest.raises(ValueError):
        eng.sample(seq, [1], 1000, params, g)
    sch = Scheduler(eng, portion=8, burst=3)
    eng.close(seq)
    both = [sch.submit(prompt, 25, sampling=params), sch.submit(prompt, 12)]
    list(sch.run())
    assert both[0].generated == tokens
    seq = eng.open()
    assert both[1].generated == eng.greedy(seq, prompt, 12)


def test_sampling_requests_do_not_depend_on_bursts(tmp_path):
    """The 4-bit decoder behind the scheduler: sampled and greedy requests side by side, the same tokens however they are dealt out."""
    (tmp_path / "config.json").write_text(json.dumps(CONFIG))
    seen = []
    for portion, burst, cache in ((8, 4, "e4m3"), (64, 16, "e4m3"), (3, 1, "e4m3"), (8, 4, "f16"), (64, 7, "f16")):
        engine = registry.load(str(tmp_path), kv_cache=cache)
        sch = Scheduler(engine, portion=portion, burst=burst)
        requests = [sch.submit([5, 9, 200], 23, sampling=SamplingParams(temperature=1.2, top_p=0.9, seed=8)), sch.submit([7], 9),
                    sch.submit([5, 9, 200], 23, sampling=SamplingParams(temperature=1.2, top_p=0.9, seed=9))]
        list(sch.run())
        seen.append([r.generated for r in requests])
    assert seen[0] == seen[1] == seen[2] and seen[3] == seen[4]
    assert seen[0][0] != seen[0][2] and all(len(r) == n for r, n in zip(seen[0], (23, 9, 23)))


def test_command_line(tmp_path, capsys):
    from tensorwarp_b200.__main__ import main
    (tmp_path / "config.json").write_text(json.dumps(CONFIG))
    base = ["generate", "--model", str(tmp_path), "--tokens", "1,2,3", "--tokens", "4", "--max-new-tokens", "8"]
    outs = []
    for more in ([], ["--temperature", "0"], ["--temperature", "1.5", "--seed", "3"], ["--temperature", "1.5", "--seed", "3"],
                 ["--temperature", "1.5", "--seed", "3", "--kv-cache", "e4m3", "--top-k", "1"]):
        assert main(base + more) == 0
        outs.append(capsys.readouterr().out)
    assert outs[0] == outs[1] and outs[2] == outs[3] and outs[2] != outs[0] and outs[4].count("\n") == 2


def test_refusals_of_the_engine(model):
    with pytest.raises(_lib.TwmError):
        QuantizedGenerationEngine(model, kv_cache="int8")
    eng = QuantizedGenerationEngine(model, kv_cache="e4m3")
    with pytest.raises(_lib.TwmError):
        eng.generate_tw_marlin_graph(1, 5, SamplingParams(), random=torch.rand(4))
    with pytest.raises(_lib.TwmError):
        eng.generate_tw_marlin_graph(1, 301, SamplingParams())
    cache = cache8.Cache8.empty(2, 64, 1, 64)
    q = torch.zeros((2, 64), dtype=torch.float16, device="cuda")
    start = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (dict(start=start[:1]), dict(start=start.long()), dict(q=q.float()), dict(q=q[:, :32]), dict(row_start=start), dict(max_rows=2), dict(num_heads=3)):
        args = {"q": q, "out": torch.zeros_like(q), "start": start, "num_heads": 1, **bad}
        with pytest.raises(_lib.TwmError):
            cache8.attention(cache, args.pop("q"), args.pop("out"), args.pop("start"), **args)
