"""Generation from the 8-bit cache (`cache_format="q8"`): a Qwen3 of heads of 64, fed whole, in portions and one token at a time,
against the plain model whose keys and values pass through the format's rounding; through `Engine`, eager and from graphs.

The yardstick is the rounding itself: F = the distance of the plain model with rounded keys and values from the plain model
without. In float32 the engine rounds the same values but for those that lie within a few 2^-20 of a boundary between two codes;
such a value moves by one step, as far as two of the others are off. Were one value in a hundred that near (it is some in a
million), the sum of their squares would be 0.01 * (2 / (1 / sqrt(3)))^2 = 0.12 of all values' squares, the root 0.35: a distance
of F / 2 holds, and a token, a head or a scale that is missed does not."""
from __future__ import annotations

import functools

import pytest
import torch

from holon_amd.config import EngineConfig, SamplingParams
from holon_amd.engine.loading import load_model
from holon_amd.kernels.continuation import ContinuationOps
from holon_amd.kernels.hip import KernelError
from tests import dopirax_models, falisun_models, helpers as H
from tests.plain import qwen3
from tests.plain.ops import TorchKernels, quantise_q8

DEVICES = [pytest.param("cpu", id="cpu-twin"), pytest.param("cuda", marks=pytest.mark.gpu, id="hip")]
LENGTHS = (40, 70, 33, 90, 1)
VOCAB = H.CONFIG_C["vocab_size"]


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return H.make_folder(tmp_path_factory.mktemp("models") / "C", H.CONFIG_C, 2, 2.0)


def _rounded(x):
    codes, byte = quantise_q8(x)
    return (codes.view(torch.float8_e4m3fn).double() * torch.exp2(byte.double() - 127)[..., None]).to(x.dtype)


@pytest.fixture(scope="module")
def logits(folder):
    """(request, dtype, rounded keys and values) -> the plain model's logits."""
    requests = {f"r{i}": H.random_ids(n, VOCAB, 100 + i) for i, n in enumerate(LENGTHS)}
    whole, found = qwen3.causal_attention, {}
    for dtype in (torch.float32, torch.bfloat16):
        plain = qwen3.PlainQwen3(folder, dtype)
        for rounded in (False, True):
            with pytest.MonkeyPatch.context() as m:
                if rounded:
                    m.setattr(qwen3, "causal_attention", lambda q, k, v, window=0: whole(q, _rounded(k), _rounded(v), window))
                found[dtype, rounded] = {r: plain.logits(list(ids)) for r, ids in requests.items()}
    return requests, found


def _replayer(folder, device, dtype, **kw):
    from holon_amd.engine.replay import Replayer
    return Replayer(load_model(folder, device=device, dtype=dtype, kernels=TorchKernels() if device == "cpu" else None,
                               page_size=kw.pop("page_size", 16), max_seqs=4, max_model_len=512, max_step_tokens=512,
                               cache_tokens=512, cache_format="q8", **kw))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("page_size", [16, 48])
def test_every_way_of_cutting(folder, logits, dtype, page_size, device):
    requests, found = logits
    rep = _replayer(folder, device, dtype, page_size=page_size)
    state = rep.cache.groups[0].storage
    assert state.dtype is torch.uint8 and state.shape[2] == page_size * 2 * 2 * 65
    traces = [H.trace_whole(requests), H.trace_decode_tail("r1", requests["r1"], 32),
              H.trace_chunks("r3", requests["r3"], [7, 2, 13, 3, 2, 30, 5]), H.trace_mixed(requests, 0)]
    for i, trace in enumerate(traces):
        got = H.run_trace(rep, trace)
        g, exact = H.gather(found[torch.float32, False], got)
        _, rounded = H.gather(found[getattr(torch, dtype), True], got)
        floor = H.rel_rms(H.gather(found[torch.float32, True], got)[1], exact)
        if dtype == "float32":
            assert torch.isfinite(g).all() and H.rel_rms(g, rounded) <= floor / 2, (i, H.rel_rms(g, rounded), floor)
        else:
            H.assert_bf16_close(g, exact, rounded, f"trace {i}")
        rep.cache.check()
    assert all(g.pool.free == g.pool.usable for g in rep.cache.groups)


def _engine(folder, device, **kw):
    from holon_amd.engine.engine import Engine
    shape = dict(dtype="float32", page_size=16, max_seqs=4, max_model_len=256, max_step_tokens=64, cache_format="q8")
    return Engine(EngineConfig(model=str(folder), device=device, **{**shape, **kw}),
                  kernels=TorchKernels() if device == "cpu" else None)


@pytest.mark.parametrize("device", DEVICES)
def test_prompts_that_start_alike_share_their_pages(folder, device):
    """The pages of a prefix are found again, by requests of the same round and of the next: the same tokens, less work."""
    start = H.random_ids(64, VOCAB, 5)
    prompts = [start + H.random_ids(n, VOCAB, 20 + n) for n in (3, 17, 30, 9)]
    params = SamplingParams(temperature=0.0, max_tokens=12, ignore_eos=True)
    alone = _engine(folder, device, prefix_cache=False)
    want = alone.generate(prompts, params)
    shared = _engine(folder, device)
    assert shared.generate(prompts, params) == want and shared.generate(prompts, params) == want
    assert shared.stats()["prefix_tokens_saved"] >= 4 * 64
    # a pool that holds little more than one request: preempted, recomputed, the same
    tight = _engine(folder, device, cache_tokens=160, max_model_len=128, prefix_cache=False)
    assert tight.generate(prompts, params) == want
    # half of the 16-bit pages' bytes, and one more a (token, head)
    plain = _engine(folder, device, cache_format="model", dtype="bfloat16")
    of = [e.cache.groups[0].storage for e in (shared, plain)]
    ratio = (of[0][0, 0].numel() * of[0].element_size()) / (of[1][0, 0].numel() * of[1].element_size())
    assert ratio == 65 / 128


@pytest.mark.gpu
def test_graph_replays_equal_eager_steps(folder):
    prompts = [H.random_ids(n, VOCAB, 80 + n) for n in (3, 17, 8, 1)]
    outs = {}
    for graphs in (False, True):
        engine = _engine(folder, "cuda", graphs=graphs)
        rids = [engine.add(p, SamplingParams(temperature=0.0 if i % 2 else 0.7, seed=5, max_tokens=20 + 7 * i,
                                             ignore_eos=True)) for i, p in enumerate(prompts)]
        got = {r: [] for r in rids}
        while engine.has_work():
            for d in engine.step():
                got[d.rid].extend(d.token_ids)
        outs[graphs] = [got[r] for r in rids]
        if graphs:
            assert engine.runner.graph_replays > 20
    assert outs[True] == outs[False]


def test_what_it_refuses():
    with pytest.raises(ValueError, match="cache_format must be one of"):
        EngineConfig(model="m", cache_format="fp8")
    kernels = TorchKernels()
    kernels.check_cache_q8 = functools.partial(ContinuationOps.check_cache_q8, kernels)
    for config, page in ((H.CONFIG_A, 16), (H.CONFIG_C, 8)):                 # heads of 16; pages of 8 tokens
        with pytest.raises(KernelError, match="8-bit cache: heads of"):
            load_model("", device="cpu", dtype="float32", kernels=kernels, page_size=page, cache_format="q8", random_config=config)
    for config in (dopirax_models.CONFIG_A, falisun_models.CONFIG_A):                # other attention keeps its own state, in its own types
        with pytest.raises(ValueError, match="cache_format q8 is served by grouped-query attention alone"):
            load_model("", device="cpu", dtype="float32", kernels=TorchKernels(), cache_format="q8", random_config=config)


def test_models_without_keys_and_values_are_refused():
    """A model that keeps nothing by token has no cache whose format could be asked for."""
    from holon_amd.registry import register_architecture, register_part, unregister_architecture, unregister_part
    from tests.toy_parts import GridRunningMean, ToyConfig, toy_recipe
    config = {"architectures": ["ToyGridModel"], "width": 48, "tokens": 61, "depth": 2, "grid": 8, "eps": 1e-5}
    register_part("mixer", "test-grid-mean")(GridRunningMean)
    register_architecture("ToyGridModel", ToyConfig, toy_recipe)
    try:
        load_model("", device="cpu", dtype="float32", kernels=TorchKernels(), random_config=config)
        with pytest.raises(ValueError, match="keeps no keys and values"):
            load_model("", device="cpu", dtype="float32", kernels=TorchKernels(), cache_format="q8", random_config=config)
    finally:
        unregister_part("mixer", "test-grid-mean")
        unregister_architecture("ToyGridModel")
