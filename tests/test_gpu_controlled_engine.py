"""Shared-prefix decode and logit controls through the engine, teacher-forced
against the CPU oracle model."""
import pytest
import torch

from oracle import model as OM
from test_gpu_engine import _engine, teacher_forced_agreement
from test_gpu_runner import CFG, _our_model

pytestmark = pytest.mark.gpu


@pytest.fixture
def weights():
    return OM.random_weights(CFG, seed=5, dtype=torch.bfloat16, std=0.2)


def prompts_of(lengths, shared=70, seed=6):
    g = torch.Generator().manual_seed(seed)
    head = torch.randint(0, CFG.vocab_size, (shared,), generator=g).tolist()
    return [head + torch.randint(0, CFG.vocab_size, (n,), generator=g).tolist() for n in lengths]


def count_calls(monkeypatch):
    """Calls of the shared-prefix attention and of its graphs' replays."""
    from tinyvllm.runtime import attention, graphs

    calls = {"kernel": 0, "replay": 0}
    kernel, replay = attention.paged_decode_shared_prefix, graphs.DecodeGraphs.replay_shared

    def counted(*args, **kwargs):
        calls["kernel"] += 1
        return kernel(*args, **kwargs)

    def replayed(self, *args):
        calls["replay"] += 1
        return replay(self, *args)

    monkeypatch.setattr(attention, "paged_decode_shared_prefix", counted)
    monkeypatch.setattr(graphs.DecodeGraphs, "replay_shared", replayed)
    return calls


@pytest.mark.parametrize("eager,kv_dtype", [(False, None), (True, None),
                                            (False, torch.float8_e4m3fn)])
def test_shared_prefix_decode_matches_oracle(device, weights, monkeypatch, eager, kv_dtype):
    from tinyvllm import GenerateRequest, SamplingParams
    from tinyvllm.runtime import runner

    monkeypatch.setattr(runner, "_SHARED_PREFIX_BYTES", 1)  # share wherever pages are common
    calls = count_calls(monkeypatch)
    scales = (0.5, 0.25) if kv_dtype is not None else (1.0, 1.0)
    engine = _engine(_our_model(weights, device), shared_prefix_attention=True,
                     enforce_eager=eager, kv_cache_dtype=kv_dtype, kv_scales=scales)
    prompts = prompts_of((3, 40, 1, 90)) + prompts_of((20,), shared=130, seed=9)
    new = 10
    params = SamplingParams(max_new_tokens=new, ignore_eos=True)
    outs = engine.generate([GenerateRequest(p, params) for p in prompts])
    agree = sum(teacher_forced_agreement(weights, p, o.output_token_ids,
                                         kv_fp8=scales if kv_dtype is not None else None)
                for p, o in zip(prompts, outs))
    assert agree / (new * len(prompts)) >= 0.99, agree
    assert calls["kernel"] if eager else calls["replay"] >= 5
    engine.close()


def test_sharing_waits_for_enough_bytes_and_leaves_the_default_alone(device, weights,
                                                                     monkeypatch):
    from tinyvllm import GenerateRequest, SamplingParams

    calls = count_calls(monkeypatch)
    params = SamplingParams(max_new_tokens=4, ignore_eos=True)
    requests = [GenerateRequest(p, params) for p in prompts_of((3, 9))]
    plain = _engine(_our_model(weights, device))
    assert plain.executor.runner.shared_prefix is None
    want = [o.output_token_ids for o in plain.generate(requests)]
    plain.close()
    assert calls == {"kernel": 0, "replay": 0}
    engine = _engine(_our_model(weights, device), shared_prefix_attention=True)
    captured = calls["kernel"]
    assert captured
    assert [o.output_token_ids for o in engine.generate(requests)] == want
    assert calls == {"kernel": captured, "replay": 0}  # tiny prefixes: not worth it
    engine.close()


def controlled_logits(row, params, prompt, answer):
    """The formula on one oracle row."""
    x = row.float().clone()
    for i in set(prompt) | set(answer):
        x[i] = x[i] / params.repetition_penalty if x[i] > 0 else x[i] * params.repetition_penalty
        k = answer.count(i)
        x[i] -= params.frequency_penalty * k + params.presence_penalty * (k > 0)
    for i, b in params.logit_bias:
        x[i] += b
    if params.allowed_token_ids is not None:
        keep = torch.zeros_like(x, dtype=torch.bool)
        keep[list(params.allowed_token_ids)] = True
        x[~keep] = float("-inf")
    return x


def greedy_agreement(weights, prompt, ours, params):
    logits = OM.forward(CFG, weights, list(prompt) + list(ours))
    agree = 0
    for i, token in enumerate(ours):
        row = logits[len(prompt) - 1 + i]
        x = controlled_logits(row, params, list(prompt), list(ours[:i]))
        # Near ties as without controls, and the changed logits' own rounding.
        scale = max(float(row.abs().max()), float(x[x.isfinite()].abs().max()))
        agree += int(x[token] >= x.max() - max(0.05, scale * 2.0 ** -6))
    return agree


@pytest.mark.parametrize("pipelined", [True, False])
@pytest.mark.parametrize("shared", [True, False])
def test_controls_match_oracle(device, weights, monkeypatch, pipelined, shared):
    """Requests with every control and with none, more of them than slots, so
    that rows of the device history pass from one request to the next."""
    from tinyvllm import GenerateRequest, SamplingParams
    from tinyvllm.runtime import runner

    monkeypatch.setattr(runner, "_SHARED_PREFIX_BYTES", 1)
    engine = _engine(_our_model(weights, device), pipelined=pipelined,
                     shared_prefix_attention=shared)
    new = 12
    common = dict(max_new_tokens=new, ignore_eos=True)
    kinds = [
        SamplingParams(**common),
        SamplingParams(repetition_penalty=1.4, **common),
        SamplingParams(frequency_penalty=100.0, **common),
        SamplingParams(presence_penalty=3.0, logit_bias={5: 40.0, 6: -40.0}, **common),
        SamplingParams(allowed_token_ids=range(32, 64), **common),
        SamplingParams(repetition_penalty=0.8, frequency_penalty=0.5,
                       allowed_token_ids=(1, 2, 3, 70, CFG.vocab_size - 1), **common),
        SamplingParams(temperature=1.0, seed=3, allowed_token_ids=(7, 8, 9), **common),
    ]
    prompts = prompts_of((3, 40, 1, 17, 5, 90, 30))
    outs = engine.generate([GenerateRequest(p, k) for p, k in zip(prompts, kinds)])
    agree = total = 0
    for prompt, params, out in zip(prompts, kinds, outs):
        ours = list(out.output_token_ids)
        assert len(ours) == new
        if params.allowed_token_ids is not None:
            assert set(ours) <= params.allowed_token_ids
        if params.frequency_penalty == 100.0:
            assert len(set(ours)) == new  # nothing twice
        if params.greedy:
            agree += greedy_agreement(weights, prompt, ours, params)
            total += new
    assert agree / total >= 0.98, (agree, total)
    # An id that comes again starts from an empty history.
    again = engine.generate([GenerateRequest(prompts[2], kinds[2])])[0]
    assert list(again.output_token_ids) == list(outs[2].output_token_ids)
    engine.close()


def test_controls_are_checked_at_submission(device, weights):
    from tinyvllm import SamplingParams

    engine = _engine(_our_model(weights, device))
    with pytest.raises(ValueError, match="vocabulary"):
        engine.submit([1, 2], SamplingParams(logit_bias={CFG.vocab_size: 1.0}))
    with pytest.raises(ValueError, match="vocabulary"):
        engine.submit([1, 2], SamplingParams(allowed_token_ids=[0, CFG.vocab_size]))
    engine.close()
