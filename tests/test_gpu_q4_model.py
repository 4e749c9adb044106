"""The target with its dense projections and its KV cache in 4 bits: against the fp64 oracle on the values
that the 4-bit tensors hold, and the promises of the full-precision path (steps equal blocks, greedy
speculative decoding equals native decoding)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import _q4_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cuda():
    from evspark_b200 import _native as N

    N.call("evs_device_check")
    return torch.device("cuda:0")


def tokens(n, seed=0):
    return np.random.default_rng(seed).choice([65, 67, 71, 84], size=n)


def held_weights(model, w):
    """The oracle's weights: what the model's 4-bit projections hold, the rest as it was."""
    out = dict(w)
    for name, q in model.q4_weights.items():
        v = q.dequantize(torch.float32).cpu()
        if name.endswith(".w1"):
            f, d = v.shape[0] // 2, v.shape[1]
            pair = v.view(f // 64, 2, 64, d)
            out[name], out[name[:-1] + "2"] = pair[:, 0].reshape(f, d), pair[:, 1].reshape(f, d)
        else:
            out[name] = v
    return out


@pytest.fixture(scope="module")
def tiny(cuda):
    from evspark_b200.config import TINY
    from evspark_b200.model import TargetModel
    from evspark_b200.weights import init_target_weights

    w = init_target_weights(TINY, seed=20260820)
    return {fmt: TargetModel(TINY, w, device=cuda, weight_format=fmt[0], kv_format=fmt[1], weight_group=32)
            for fmt in (("q4", None), (None, "q4"), ("q4", "q4"))}, w


def test_q4_weights_match_the_oracle_on_the_held_values(tiny):
    """fp32 model: logits within the fp32 path's bound (1e-5) of the fp64 oracle on the held weights."""
    from evspark_b200.config import TINY
    from evspark_b200.specdec.block import block_forward, prefill, slice_states_to_accept
    from oracle.model import OracleTarget

    models, w = tiny
    model = models["q4", None]
    assert not any(n.rsplit(".", 1)[-1] in ("w_in", "w_o", "w1", "w2", "w3") for n in model.weights)
    o = OracleTarget(TINY, held_weights(model, w))
    prompt, chunk = tokens(64), tokens(13, 1)
    ip, st = model.initialize_inference_params(128), o.init_state(1, 128)
    p = prefill(model, torch.as_tensor(prompt)[None], ip)
    po, _, _ = o.forward(prompt[None], st, prefill=True)
    assert float((p.cpu().double().reshape(-1) - po[:, -p.shape[1]:].reshape(-1)).abs().max()) <= 1e-5
    logits, stash = block_forward(model, torch.as_tensor(chunk)[None], ip, retain=True)
    ref, so, _ = o.forward(chunk[None], st, retain=True)
    assert float((logits.cpu().double() - ref).abs().max()) <= 1e-5
    slice_states_to_accept(ip, stash, 4)
    o.slice(st, so, 4)
    again = model(torch.as_tensor(chunk[:3])[None], inference_params_dict=ip)[0]
    ref, _, _ = o.forward(chunk[None, :3], st)
    assert float((again.cpu().double() - ref).abs().max()) <= 1e-5
    ip.close()


@pytest.mark.parametrize("fmt", [(None, "q4"), ("q4", "q4")])
def test_q4_cache_holds_the_oracles_keys_and_feeds_its_attention(tiny, fmt):
    """The cache's values are the oracle's keys and values in the format (a code may differ only where the
    oracle's fp64 quotient is a half to within the fp32 model's own error), and the oracle's attention over
    them gives the logits."""
    from evspark_b200.config import TINY
    from evspark_b200.specdec.block import block_forward, prefill
    from oracle.model import OracleTarget

    models, w = tiny
    model = models[fmt]
    prompt, chunk = tokens(100, 2), tokens(13, 3)
    L, n = len(prompt), len(prompt) + len(chunk)
    ip = model.initialize_inference_params(160)
    prefill(model, torch.as_tensor(prompt)[None], ip)
    logits = block_forward(model, torch.as_tensor(chunk)[None], ip)
    kv = ip.export(3, 3, kv_len=n)[0].cpu().double()  # [n, 2, H, Dh]
    seen = []

    class Held(OracleTarget):
        def rope(self, x, pos):
            out = super().rope(x, pos)
            seen.append(out)
            return out

        def _mha(self, i, a, st):
            cfg = self.cfg
            B, T, d = a.shape
            qkv = self.q(a @ self.w[f"blocks.{i}.w_qkv"].T).view(B, T, 3, cfg.n_heads, cfg.head_dim)
            L0 = int(st.lengths[0])
            pos = torch.arange(L0, L0 + T)
            q, k = self.rope(qkv[0, :, 0], pos), self.rope(qkv[0, :, 1], pos)
            for got, want in ((kv[L0:L0 + T, 0], k), (kv[L0:L0 + T, 1], qkv[0, :, 2])):
                c, s = R.quantize(want, 32)
                sc = s.repeat_interleave(32, -1)
                ratio = want / sc
                # fp32 activations of this model are within 1e-5 of the oracle's (the test above): the
                # scales are theirs or, at a rounding border, a 1/16 off; codes differ near halves alone
                off = (got / sc - (c - 8)).abs() > 1e-9
                half = ((ratio - ratio.floor()) - 0.5).abs() < 1e-3
                m, _ = torch.frexp(want.unflatten(-1, (-1, 32)).abs().amax(-1) / 7)
                border = ((m * 32) % 1 - 0.5).abs() < 1e-2
                assert not bool((off & ~half & ~border.repeat_interleave(32, -1)).any())
                assert float(off.double().mean()) < 1e-2
            out, _, _ = R.attend(q, kv[:L0 + T, 0], kv[:L0 + T, 1], L0, cfg.head_dim ** -0.5)
            return out.reshape(1, T, d)

    o = Held(TINY, held_weights(model, w))
    st = o.init_state(1, 160)
    o.forward(prompt[None], st, prefill=True)
    ref, _, _ = o.forward(chunk[None], st)
    assert float((logits.cpu().double() - ref).abs().max()) <= 1e-5
    assert L == 100
    ip.close()


@pytest.mark.parametrize("fmt", [("q4", None), (None, "q4"), ("q4", "q4")])
def test_blocks_steps_chunks_rollback_and_rows_agree_bit_for_bit(tiny, fmt):
    from evspark_b200.specdec.block import block_forward, prefill, slice_states_to_accept

    models, _ = tiny
    model = models[fmt]
    prompt, chunk = torch.as_tensor(tokens(90, 4))[None], torch.as_tensor(tokens(13, 5))[None]
    ip = model.initialize_inference_params(200, max_batch=3)
    prefill(model, prompt, ip)
    step = ip.clone()
    block, stash = block_forward(model, chunk, ip, retain=True)
    # prefill in other chunks, and the block one token at a time.  Projections of an fp32 model without
    # 4-bit weights split their sums by shape alone too, so every format keeps its bits.
    small = model.initialize_inference_params(200, max_batch=3, max_chunk=16)
    prefill(model, prompt, small)
    assert torch.equal(block_forward(model, chunk, small), block)
    for t in range(13):
        assert torch.equal(model(chunk[:, t:t + 1], inference_params_dict=step)[0][:, 0], block[:, t]), t
    slice_states_to_accept(ip, stash, 6)
    twin = ip.clone()
    ip.expand(3)
    three = ip.forward(chunk.repeat(3, 1))
    one = twin.forward(chunk)
    assert torch.equal(three[0], one[0]) and torch.equal(three[2], one[0])
    ip.collapse(2)
    assert torch.equal(ip.forward(chunk[:, :4]), twin.forward(chunk[:, :4]))
    assert ip.device_error() == (0, 0, 0)
    for x in (ip, step, small, twin):
        x.close()


def test_bf16_speculative_equals_native(cuda):
    """7B width, every block kind: greedy speculative decoding with a neural drafter equals native decoding."""
    from evspark_b200.api import EvSpark

    prompt = "".join(np.random.default_rng(3).choice(list("ACGT"), size=300))
    with EvSpark.load(ckpt=None, model_name="evo2_7b_slice", weight_format="q4", kv_format="q4", weight_group=64) as es:
        spec = es.generate(prompt, n_tokens=48, greedy=True)
        native = es.generate_native(prompt, n_tokens=48, greedy=True)
        assert spec.ids.tolist() == native.ids.tolist()
        assert es.generate(prompt, n_tokens=32, seed=5).ids.shape == (32,)


def test_bf16_speculative_equals_native_behind_a_long_prompt(cuda):
    """A prompt whose long chunks take the tensor-core attention: blocks and steps behind it still agree."""
    from evspark_b200.api import EvSpark

    prompt = "".join(np.random.default_rng(4).choice(list("ACGT"), size=4500))
    with EvSpark.load(ckpt=None, model_name="evo2_7b_slice", kv_format="q4", max_chunk=1024) as es:
        spec = es.generate(prompt, n_tokens=24, greedy=True)
        native = es.generate_native(prompt, n_tokens=24, greedy=True)
        assert spec.ids.tolist() == native.ids.tolist()


def test_streams_equal_single_streams(tiny):
    from evspark_b200.specdec.block import prefill

    model = tiny[0]["q4", "q4"]
    ids = torch.as_tensor(np.stack([tokens(70, s) for s in range(3)]))
    ip = model.initialize_inference_params(120, max_batch=3)
    prefill(model, ids, ip)
    nxt = torch.as_tensor(np.stack([tokens(5, 10 + s) for s in range(3)]))
    out = ip.forward(nxt)
    for b in range(3):
        one = model.initialize_inference_params(120)
        prefill(model, ids[b:b + 1], one)
        assert torch.equal(one.forward(nxt[b:b + 1])[0], out[b])
        one.close()
    ip.close()


def test_refusals(cuda):
    from evspark_b200 import _native as N
    from evspark_b200.config import TINY
    from evspark_b200.model import TargetModel
    from evspark_b200.weights import init_target_weights

    w = init_target_weights(TINY, seed=1)
    for kw in (dict(weight_format="int4"), dict(kv_format="fp8"), dict(weight_format="q4", weight_group=48),
               dict(weight_format="q4", tp=(0, 2)), dict(kv_format="q4", tp=(0, 2))):
        with pytest.raises(ValueError):
            TargetModel(TINY, w, device=cuda, **kw)
    m = TargetModel(TINY, w, device=cuda, weight_format="q4")
    q = next(iter(m.q4_weights.values()))
    assert N.lib().evs_model_set_q4(m.handle, 0, N.SLOTS["w_in"], q.codes.data_ptr(), q.scales.data_ptr(), *q.shape,
                                    q.group) == N.EVS_EINVAL  # finalized
    # states of the two cache formats do not copy into each other
    a, b = TargetModel(TINY, w, device=cuda), TargetModel(TINY, w, device=cuda, kv_format="q4")
    x, y = a.initialize_inference_params(64), b.initialize_inference_params(64)
    assert N.lib().evs_state_copy(x.handle, y.handle, None) == N.EVS_EINVAL
    x.close(), y.close()
