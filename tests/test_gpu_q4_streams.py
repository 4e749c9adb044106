"""The 4-bit formats behind long prompts: a state does not depend on the chunks in which its prompt was prefilled,
so batched streams, candidates and teacher-forced states agree with single decoding as they do in bf16."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

LONG = 4300  # bf16, head_dim 128: prompt positions from 4,096 on take the tcgen05 attention
FORMATS = [(None, "q4"), ("q4", "q4")]


def prompts(rows, length, seed):
    return np.stack([np.random.default_rng(seed + b).choice([65, 67, 71, 84], size=length)
                     for b in range(rows)]).astype(np.int64)


@pytest.fixture(scope="module", params=FORMATS, ids=["kv", "weights+kv"])
def slice7b(request):
    """Four blocks of 7B width, attention before and behind others (a difference of its sums reaches the states
    of the later blocks), with a drafter for three rows."""
    from evspark_b200.config import DRAFTERS, EVO2_7B_SLICE, HCL, HCM, MHA
    from evspark_b200.drafter import DeviceDrafter, layer_index
    from evspark_b200.model import TargetModel
    from evspark_b200.specdec.block.neural_draft import NeuralDraftModel

    dcfg = DRAFTERS["evo2_7b_slice"]
    cfg = EVO2_7B_SLICE.with_(layer_types=(HCM, MHA, HCL, MHA))
    model = TargetModel.random(cfg, seed=11, device="cuda:0", init_on="cuda", weight_format=request.param[0],
                               kv_format=request.param[1],
                               capture_layers=tuple(layer_index(x) for x in dcfg.inject_layers))
    dr = DeviceDrafter.random(dcfg, embed=model.weights["embed"], device="cuda:0", max_batch=3, init_on="cuda")
    nd = NeuralDraftModel(model, dr, dcfg.inject_layers)
    yield model, nd
    nd.close()
    model.close()


def test_prefill_does_not_depend_on_its_chunks(slice7b):
    from evspark_b200.specdec.block import block_forward, prefill

    model, _ = slice7b
    ids, chunk = (torch.as_tensor(prompts(1, n, s)) for n, s in ((LONG, 1), (13, 2)))
    seen = []
    for max_chunk in (1024, 32, 100):
        ip = model.initialize_inference_params(LONG + 40, max_chunk=max_chunk)
        last = prefill(model, ids, ip)[:, -1]
        seen.append((last, ip.export(1, 3), ip.export(2, 2), ip.export(3, 3), block_forward(model, chunk, ip)))
        assert ip.device_error() == (0, 0, 0)
        ip.close()
    for other in seen[1:]:
        for a, b in zip(seen[0], other):
            assert torch.equal(a, b)


def test_forwards_of_any_length_equal_steps(slice7b):
    """A forward of more than 64 tokens behind a long prompt, too."""
    from evspark_b200.specdec.block import prefill

    model, _ = slice7b
    ids, more = (torch.as_tensor(prompts(1, n, s)) for n, s in ((LONG, 3), (70, 4)))
    ip = model.initialize_inference_params(LONG + 80, max_chunk=128)
    prefill(model, ids, ip)
    steps = ip.clone()
    block = ip.forward(more)
    for t in range(more.shape[1]):
        assert torch.equal(steps.forward(more[:, t:t + 1])[:, 0], block[:, t]), t
    ip.close(), steps.close()


@pytest.mark.parametrize("length", [80, LONG])
def test_streams_equal_single_decoding(slice7b, length):
    from evspark_b200.specdec.block.loop import native_greedy_reference, speculative_generate
    from evspark_b200.specdec.block.streams import speculative_generate_streams

    model, nd = slice7b
    B, n = 3, 16
    p = prompts(B, length, 300)
    nd.capture_reset()
    res = speculative_generate_streams(model, nd, p, n, 12, True, [np.random.default_rng(0)] * B)
    for b in range(B):
        nat, ip, _ = native_greedy_reference(model, torch.as_tensor(p[b])[None], n)
        ip.close()
        np.testing.assert_array_equal(res.emitted[b], nat, err_msg=f"greedy stream {b}")
    res.inference_params_dict.close()
    nd.capture_reset()
    res = speculative_generate_streams(model, nd, p, n, 12, False, [np.random.default_rng(s) for s in range(B)])
    for b in range(B):
        nd.capture_reset()
        one = speculative_generate(model, nd, torch.as_tensor(p[b])[None], n, 12, greedy=False,
                                   rng=np.random.default_rng(b))
        np.testing.assert_array_equal(res.emitted[b], one.emitted_ids, err_msg=f"sampled stream {b}")
        one.inference_params_dict.close()
    res.inference_params_dict.close()


def test_end_state_equals_the_teacher_forced_one(slice7b):
    from evspark_b200.specdec.block.loop import spec_end_kv_len, speculative_generate, teacher_force_to_spec_state

    model, nd = slice7b
    p, n = torch.as_tensor(prompts(1, LONG, 40)), 20
    nd.capture_reset()
    spec = speculative_generate(model, nd, p, n, 12, greedy=True, rng=np.random.default_rng(0))
    kv = spec_end_kv_len(LONG, n)
    ref = teacher_force_to_spec_state(model, p, spec.emitted_ids)
    mine = spec.inference_params_dict
    assert mine.offset == ref.offset == kv
    for layer in (1, 3):
        assert torch.equal(mine.export(layer, 3, kv_len=kv), ref.export(layer, 3, kv_len=kv))
    assert torch.equal(mine.export(2, 2), ref.export(2, 2))
    nxt = torch.as_tensor(spec.emitted_ids[-1:])[None]
    assert torch.equal(mine.forward(nxt), ref.forward(nxt))
    mine.close(), ref.close()


def test_candidates_equal_native_decoding(slice7b):
    """Three candidates a round: the state is expanded, the winner's row kept."""
    from evspark_b200.specdec.block.loop import native_greedy_reference, speculative_generate

    model, nd = slice7b
    for length in (90, LONG):
        p, n = torch.as_tensor(prompts(1, length, 50)), 12
        nat, ip, _ = native_greedy_reference(model, p, n)
        ip.close()
        nd.capture_reset()
        spec = speculative_generate(model, nd, p, n, 12, greedy=True, rng=np.random.default_rng(0), n_candidates=3)
        np.testing.assert_array_equal(spec.emitted_ids, nat)
        spec.inference_params_dict.close()
