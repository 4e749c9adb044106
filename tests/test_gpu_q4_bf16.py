"""The bf16 target in 4 bits against the oracle, block by block on the device's own residual stream: prompts run on
the decoded weights and, from position 4,096 on, on the tcgen05 attention; blocks behind them on the 4-bit linear and
the row-tile attention."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import _parity
from tests import _q4_ref as R
from tests.test_gpu_q4_model import held_weights

pytestmark = pytest.mark.gpu


def small(d, heads, inner):
    from evspark_b200.config import HCL, HCM, HCS, MHA, EVO2_7B

    kinds = (HCS, MHA, HCL, MHA) if heads == 2 else (HCM, MHA, HCS, MHA)
    return EVO2_7B.with_(name=f"bf16_{d}", d_model=d, n_layers=4, layer_types=kinds, n_heads=heads, head_dim=128,
                         mlp_inner=inner)


def oracle_blocks(cfg, weights, segs, caches):
    """Every block on its own input segments; attention over the keys and values that the device holds."""
    from oracle.model import OracleTarget

    class Held(OracleTarget):
        kv = None

        def _mha(self, i, a, st):
            if self.kv is None:
                return super()._mha(i, a, st)
            c, T, L0 = self.cfg, a.shape[1], int(st.lengths[0])
            qkv = self.q(a @ self.w[f"blocks.{i}.w_qkv"].T).view(T, 3, c.n_heads, c.head_dim)
            pos = torch.arange(L0, L0 + T)
            for what, x in enumerate((R.rotate(qkv[:, 1], pos), qkv[:, 2])):
                got = self.kv[L0:L0 + T, what]
                # half a step of the scale (1/32 more than absmax / 7 at most, and the oracle's own absmax may be a
                # bf16 step off), and the oracle's qkv, which may be a bf16 step (2^-7) off in either of a pair
                top = x.unflatten(-1, (-1, 32)).abs().amax(-1).repeat_interleave(32, -1)
                pair = qkv[:, 1 + what].abs().unflatten(-1, (2, -1)).sum(-2).repeat(1, 1, 2)
                assert bool(((got - x).abs() <= 0.5 * top / 7 * (1 + 1 / 32) * (1 + 2.0 ** -7)
                             + 2.0 ** -7 * pair).all())
            q = self.q(R.rotate(qkv[:, 0], pos))
            k, v = self.kv[:L0 + T, 0], self.kv[:L0 + T, 1]
            sc = torch.einsum("thd,lhd->htl", q, k) * c.head_dim ** -0.5
            sc = sc.masked_fill(torch.arange(L0 + T)[None, None, :] > pos[None, :, None], float("-inf"))
            return self.q(torch.einsum("htl,lhd->thd", torch.softmax(sc, -1), v).reshape(1, T, -1))

    for i in range(cfg.n_layers):
        sub = cfg.with_(name="one", n_layers=1, layer_types=(cfg.layer_types[i],))
        o = Held(sub, {f"blocks.0.{k}": v for k, v in _parity.layer_weights(weights, i).items()}, emulate=True)
        o.kv = caches.get(i)
        st = o.init_state(1, sum(x.shape[1] for x in segs[i]))
        outs = []
        for j, x in enumerate(segs[i]):
            outs.append(o.block(0, x.double(), st, prefill=j == 0))
            st.lengths = st.lengths + x.shape[1]
        yield torch.cat(outs, 1)[0]


@pytest.mark.parametrize("fmt", [("q4", None), (None, "q4"), ("q4", "q4")])
@pytest.mark.parametrize("d,heads,inner,length", [(512, 4, 1408, 600), (256, 2, 704, 4200)])
def test_blocks_match_the_oracle_on_the_held_values(d, heads, inner, length, fmt):
    from evspark_b200.model import TargetModel
    from evspark_b200.specdec.block import block_forward, prefill
    from evspark_b200.weights import init_target_weights
    from oracle.model import OracleTarget

    cfg = small(d, heads, inner)
    w = init_target_weights(cfg, seed=5)
    model = TargetModel(cfg, w, device="cuda:0", capture_layers=(0, 1, 2, 3), weight_format=fmt[0], kv_format=fmt[1])
    ids = np.random.default_rng(6).choice([65, 67, 71, 84], size=length + 13)
    ip = model.initialize_inference_params(length + 20, max_chunk=length)
    pre = prefill(model, torch.as_tensor(ids[:length])[None], ip)[0].cpu()
    blk = block_forward(model, torch.as_tensor(ids[length:])[None], ip)[0].cpu()
    xs = [_parity.capture_rows(ip, j, length + 13).cpu() for j in range(4)]
    caches = {i: ip.export(i, 3)[0].cpu().double() for i in (1, 3)} if fmt[1] else {}
    assert ip.device_error() == (0, 0, 0)
    ip.close()
    model.close()
    weights = held_weights(model, w)
    head = OracleTarget(cfg.with_(n_layers=1, layer_types=("mha",)),
                        {"embed": w["embed"], "final_norm": w["final_norm"]}, emulate=True)
    stream = [head.embed(ids[None]).float()[0]] + xs
    segs = [[x[None, :length], x[None, length:]] for x in stream[:4]]
    for i, out in enumerate(oracle_blocks(cfg, weights, segs, caches)):
        delta, own = xs[i].double() - out, xs[i].double() - stream[i].double()
        for part in (slice(0, length), slice(length, None)):  # the prompt, and the block behind it
            worst = float(delta[part].abs().max() / own[part].abs().max())
            rms = float(delta[part].pow(2).mean().sqrt() / own[part].pow(2).mean().sqrt())
            assert worst <= _parity.TOL_BLOCK_MAX and rms <= _parity.TOL_BLOCK_RMS, (i, part, worst, rms)
    ref = head.head(xs[-1].double()[None])[0]
    assert float((torch.cat([pre, blk]).double() - ref).abs().max()) <= _parity.TOL_BF16_LOGITS
