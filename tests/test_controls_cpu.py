"""Logit controls on the host: request parameters, batches, refusals."""
import dataclasses
import math

import pytest
import torch

from tinyvllm import SamplingParams
from tinyvllm.kernels._extension import load_kernels


def test_params_normalise_and_compare():
    a = SamplingParams(logit_bias={7: 1, 3: -2.5}, allowed_token_ids=[3, 7, 3])
    assert a.logit_bias == ((3, -2.5), (7, 1.0)) and a.allowed_token_ids == frozenset((3, 7))
    assert a == SamplingParams(logit_bias=((7, 1.0), (3, -2.5)), allowed_token_ids=(7, 3))
    assert hash(a) == hash(dataclasses.replace(a))
    assert a.controlled and not a.penalised
    assert sorted(a.control_token_ids) == [3, 3, 7, 7]
    plain = SamplingParams()
    assert not plain.controlled and plain.control_token_ids == ()
    assert SamplingParams(presence_penalty=0.1).penalised
    assert SamplingParams(allowed_token_ids=5).allowed_token_ids == frozenset((5,))


@pytest.mark.parametrize("wrong,error", [
    (dict(repetition_penalty=0.0), ValueError), (dict(repetition_penalty=-1.0), ValueError),
    (dict(repetition_penalty=math.inf), ValueError), (dict(presence_penalty=math.nan), ValueError),
    (dict(frequency_penalty="1"), TypeError), (dict(frequency_penalty=True), TypeError),
    (dict(presence_penalty=1e39), ValueError),  # infinite in float32
    (dict(logit_bias={-1: 1.0}), ValueError), (dict(logit_bias={1.0: 1.0}), TypeError),
    (dict(logit_bias={1: math.nan}), ValueError), (dict(logit_bias={1: "x"}), TypeError),
    (dict(allowed_token_ids=()), ValueError), (dict(allowed_token_ids=[-1]), ValueError),
    (dict(allowed_token_ids="12"), TypeError),
])
def test_params_are_checked(wrong, error):
    with pytest.raises(error):
        SamplingParams(**wrong)


def test_penalties_that_vanish_in_float32_are_refused():
    """The kernel divides by the penalty in float32: 1e-46 would be 0 there."""
    for value in (1e-46, 2.0 ** -150, 1e-39):
        with pytest.raises(ValueError, match="positive"):
            SamplingParams(repetition_penalty=value)
    assert SamplingParams(repetition_penalty=2.0 ** -126).penalised


def entry_args(**over):
    """Arguments of tvllm_logit_controls with no rows."""
    args = dict(logits=None, rows=0, vocab=100, stride=100, rep=None, pres=None, freq=None,
                history=None, num_slots=0, capacity=0, slots=None, lengths=None, prompts=None,
                newest=None, bias_tokens=None, bias_values=None, bias_offsets=None, num_bias=0,
                mask=None, mask_count=0, mask_stride=0, mask_rows=None, out=None, out_stride=100,
                dtype=0, out_dtype=0, stream=None)
    args.update(over)
    return list(args.values())


def test_entry_point_refuses_wrong_arguments():
    lib = load_kernels()
    assert lib.tvllm_logit_controls(*entry_args()) == 0
    ptr = 1 << 20
    for over, message in (
            (dict(dtype=3), b"float16, bfloat16 or float32"), (dict(out_dtype=1), b"output"),
            (dict(vocab=0), b"sizes"), (dict(rows=-1), b"sizes"), (dict(stride=99), b"overlap"),
            (dict(out_stride=99), b"overlap"), (dict(capacity=-1), b"negative"),
            (dict(capacity=1 << 31), b"history"),
            (dict(mask_rows=ptr, mask_count=1, mask_stride=3), b"bit for every token"),
            (dict(rows=1), b"null pointer"),
            (dict(rows=1, logits=ptr, out=ptr, out_dtype=2), b"in place"),
            (dict(rows=1, logits=ptr, out=ptr, out_stride=101), b"in place"),
            (dict(rows=1, logits=ptr, out=ptr, history=ptr), b"null pointer"),
            (dict(rows=1, logits=ptr, out=ptr, bias_offsets=ptr, num_bias=1), b"null pointer"),
            (dict(rows=1, logits=ptr, out=ptr, mask_rows=ptr, mask_count=1, mask_stride=4),
             b"null pointer"),
            (dict(rows=1 << 40, logits=ptr, out=ptr), b"grid")):
        assert lib.tvllm_logit_controls(*entry_args(**over)) == -1, over
        assert message in lib.tvllm_last_error(), (over, lib.tvllm_last_error())
    assert lib.tvllm_logit_controls(*entry_args()) == 0 and lib.tvllm_last_error() == b""


def test_entry_point_refuses_outputs_that_overlap_the_logits():
    lib = load_kernels()
    ptr = 1 << 20  # fp32 out of bf16 logits of 100 tokens
    base = dict(rows=4, logits=ptr, dtype=0, out_dtype=2)
    for stride, out_stride, offset in (
            (100, 100, 200), (100, 100, -200), (100, 100, 799), (100, 100, -1599),
            (600, 300, 196), (600, 300, 804)):
        args = entry_args(**base, stride=stride, out_stride=out_stride, out=ptr + offset)
        assert lib.tvllm_logit_controls(*args) == -1
        assert b"not overlap" in lib.tvllm_last_error(), (offset, lib.tvllm_last_error())
    assert lib.tvllm_logit_controls(*entry_args()) == 0


def test_batches_carry_the_histories_of_controlled_requests():
    from tinyvllm.batch import BatchBuilder, StepPlan, WorkItem
    from tinyvllm.request import RequestState, WorkClass

    import numpy as np

    class KV:
        plan_id, block_size, num_blocks = 4, 16, 8

        def __init__(self, ids):
            self.request_ids = ids

        def append_metadata(self, request_id, start, count):
            return np.array([request_id]), request_id * 16 + np.arange(start, start + count)

    def prepare(samplings):
        requests = tuple(RequestState(i, i, [1, 2, 3], s, 0, output_token_ids=[4])
                         for i, s in enumerate(samplings))
        items = tuple(WorkItem(i, i, WorkClass.DECODE, 3, 1, 3, True)
                      for i in range(len(samplings)))
        return BatchBuilder(max_model_len=16).prepare(
            StepPlan(4, items), requests, kv=KV(tuple(range(len(samplings)))))

    assert prepare([SamplingParams()] * 2).sample_histories is None
    batch = prepare([SamplingParams(), SamplingParams(presence_penalty=1.0)])
    assert batch.sample_histories == (None, ([1, 2, 3], [4]))


def test_runner_checks_controlled_batches():
    from test_runner_validate import _batch, _Cache, _runner

    plain = _batch([[3, 9], [4, 10]], befores=[6, 5], qlens=[1, 2])
    params = (SamplingParams(), SamplingParams(presence_penalty=1.0))
    history = ([1, 2], [3])
    for histories in (None, (None,), (None, None), (history, None)):
        with pytest.raises(ValueError, match="histories"):
            _runner()._validate(dataclasses.replace(
                plain, sampling_params=params, sample_histories=histories), _Cache)
    _runner()._validate(dataclasses.replace(
        plain, sampling_params=params, sample_histories=(None, history)), _Cache)
    beyond = (SamplingParams(), SamplingParams(logit_bias={100: 1.0}))
    with pytest.raises(ValueError, match="vocabulary"):
        _runner()._validate(dataclasses.replace(
            plain, sampling_params=beyond, sample_histories=(None, history)), _Cache)


def test_plain_sampler_refuses_controls():
    from tinyvllm.sampling import Sampler

    with pytest.raises(ValueError, match="tokens"):
        Sampler().sample(torch.zeros(1, 10), [SamplingParams(presence_penalty=1.0)], [0])
