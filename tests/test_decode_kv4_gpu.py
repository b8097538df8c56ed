"""Generation with a 4-bit decode cache and with sampling, on the tiny model.

The 4-bit run is compared with a bf16 run whose caches are made to hold the
values that the 4 bits stand for (the prefix before the first step, every
appended slot after its append), so that only rounding points differ: one
bf16 rounding of the rotated k instead of the eager ops' several, which can
move a code by one (a step is a fifteenth of a group's range). Logits per step
within the generation tests' tolerance, max-abs 0.15 and cosine 0.998.
"""
import importlib.util
import os

import numpy as np
import pytest
import torch

from tests.test_sample_gpu import check_rows
from tokengate_b200 import decode, ops
from tokengate_b200.decode import Sampling, generate_batch
from tokengate_b200.gate import LinLogSigGate, synthetic_e2e_gate
from tokengate_b200.inference import TokenGateModel, with_state_span
from tokengate_b200.kv4 import KV4Cache
from tokengate_b200.model import patch_model

pytestmark = pytest.mark.gpu

GOLD = os.path.join(os.path.dirname(__file__), "golden")


def _mg():
    spec = importlib.util.spec_from_file_location("make_golden", os.path.join(GOLD, "make_golden.py"))
    mg = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mg)
    return mg


def _model(cuda, e2e):
    mg = _mg()
    model = (mg.tiny_e2e_model() if e2e else mg.tiny_model()).to(cuda).to(torch.bfloat16).eval()
    patch_model(model)
    gate = synthetic_e2e_gate(model, 1, device=cuda) if e2e else LinLogSigGate(512).to(cuda)
    return model, gate


def _prompts(seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (300, 233)], [20, 10], [280, 200]


def _through_4_bits(kb, vb, start, n):
    c = KV4Cache(kb.shape[0], n, kb.shape[2], device=kb.device)
    ops.kv4_write(c, kb[:, start:start + n], vb[:, start:start + n])
    k, v = ops.kv4_read(c)
    kb[:, start:start + n].copy_(k)
    vb[:, start:start + n].copy_(v)


@pytest.mark.parametrize("e2e", [False, True])
@pytest.mark.parametrize("prune", [False, True])
def test_kv4_decode_is_the_decode_over_its_values(cuda, monkeypatch, e2e, prune):
    model, gate = _model(cuda, e2e)
    prompts, starts, ends = _prompts(31)
    steps = 7
    forced = torch.randint(0, 1000, (2, steps - 1), generator=torch.Generator().manual_seed(5))

    def run(**kw):
        lg = []
        r = generate_batch(model, gate, prompts, starts, ends, 1, 30, steps, forced_tokens=forced, logits_out=lg,
                           prune_below_gate=prune, **kw)
        torch.cuda.synchronize()
        assert ops.device_error() == 0 and r.steps == steps - 1
        return torch.stack(lg)

    got = run(kv_bits=4)
    assert torch.equal(got, run(kv_bits=4, use_graph=False))

    made = decode._DecodeCache

    class Held(made):
        def __init__(self, cache, n_layers, extra):
            super().__init__(cache, n_layers, extra)
            for kb, vb, w in zip(self.k, self.v, self.width):
                _through_4_bits(kb, vb, 0, w)

    append = ops.qk_norm_rope_append

    def held_append(*a):
        append(*a)
        _through_4_bits(a[8], a[9], int(a[10]), 1)

    monkeypatch.setattr(decode, "_DecodeCache", Held)
    monkeypatch.setattr(ops, "qk_norm_rope_append", held_append)
    ref = run(use_graph=False)
    err = (got - ref).abs().max().item()
    cos = torch.nn.functional.cosine_similarity(got.flatten(), ref.flatten(), dim=0).item()
    assert err <= 0.15 and cos >= 0.998, (err, cos)


def test_what_four_bits_cost_a_generation(cuda):
    """Logits of a bf16 and of a 4-bit decode cache on the tiny model: an attention output over some 100 to 300 keys
    moves by about a tenth (test_what_four_bits_cost), in each of at most four layers, and is a part of the residual
    stream: within 0.4 of the logits' size, cosine above 0.92."""
    model, gate = _model(cuda, False)
    prompts, starts, ends = _prompts(33)
    forced = torch.randint(0, 1000, (2, 8), generator=torch.Generator().manual_seed(6))
    lg = {}
    for bits in (16, 4):
        lg[bits] = []
        generate_batch(model, gate, prompts, starts, ends, 1, 30, 9, forced_tokens=forced, logits_out=lg[bits], kv_bits=bits)
    a, b = torch.stack(lg[16]).double(), torch.stack(lg[4]).double()
    rel = ((a - b).norm() / a.norm()).item()
    cos = torch.nn.functional.cosine_similarity(a.flatten(), b.flatten(), dim=0).item()
    print(f"logits: relative difference {rel:.4f}, cosine {cos:.5f}")
    assert 0 < rel <= 0.4 and cos >= 0.92 and len(model.model.layers) <= 4


def test_sampled_tokens_follow_the_logits(cuda):
    """Every drawn token is the definition's for its step's logits and uniform number, eager and as a graph;
    one seed gives one text, greedy settings give the greedy text."""
    model, gate = _model(cuda, False)
    prompts, starts, ends = _prompts(32)
    steps, B = 9, 2
    settings = dict(temperature=[0.9, 1.4], top_k=[40, 0], top_p=0.95, min_p=None)

    def run(seed, **kw):
        lg = []
        gen = torch.Generator(device=cuda).manual_seed(seed)
        r = generate_batch(model, gate, prompts, starts, ends, 1, 30, steps, logits_out=lg,
                           sampling=Sampling(generator=gen, **{**settings, **kw}))
        return r, lg

    r, lg = run(1)
    u = torch.rand((steps, B), dtype=torch.float32, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).cpu().numpy()
    full = lambda v: np.broadcast_to(np.asarray(v, dtype=np.float32), (B,))  # noqa: E731
    for s in range(steps - 1):
        check_rows(lg[s].cpu().numpy(), u[s + 1], full(settings["temperature"]), np.array(settings["top_k"]), full(0.95), full(0.0),
                   np.array([t[s + 1] for t in r.token_ids]), np.array([p[s + 1] for p in r.logprobs]))
    assert all(len(t) == len(p) == steps for t, p in zip(r.token_ids, r.logprobs))
    assert run(1)[0].token_ids == r.token_ids and run(2)[0].token_ids != r.token_ids
    greedy = generate_batch(model, gate, prompts, starts, ends, 1, 30, steps)
    assert greedy.logprobs is None
    for kw in (dict(temperature=0.0), dict(temperature=1.0, top_k=1)):
        g, _ = run(3, **kw)
        assert g.token_ids == greedy.token_ids and all(p == 0 for row in g.logprobs for p in row)


def test_generate_api(cuda):
    model, gate = _model(cuda, False)
    tm = TokenGateModel(model, gate, 1, "tiny")
    ids = with_state_span(list(range(5)), list(range(100, 400)), list(range(7)))
    kw = dict(max_kept_prefill_tokens=25, max_new_tokens=6)
    plain = tm.generate(ids, None, **kw)
    assert plain.logprobs is None
    four = tm.generate(ids, None, kv_bits=4, **kw)
    assert four.token_ids[0][0] == plain.token_ids[0][0] and len(four.token_ids[0]) == 6
    draw = lambda **k: tm.generate(ids, None, generator=torch.Generator(device=cuda).manual_seed(4), **{**kw, **k})  # noqa: E731
    a = draw(temperature=1.5, top_p=0.9, min_p=0.01, kv_bits=4)
    assert a.token_ids == draw(temperature=1.5, top_p=0.9, min_p=0.01, kv_bits=4).token_ids
    one = draw(temperature=1.5, top_p=0.9, min_p=0.01, max_new_tokens=1)
    assert len(one.token_ids[0]) == len(one.logprobs[0]) == 1
    for bad in (dict(top_k=3), dict(top_p=0.5), dict(min_p=0.1), dict(kv_bits=8), dict(temperature=[1.0, 2.0]),
                dict(temperature=float("nan"))):
        with pytest.raises(ValueError):
            tm.generate(ids, None, **bad, **kw)
    with pytest.raises(ValueError):
        generate_batch(model, gate, [list(range(50))], [5], [40], 1, 5, 3, kv_bits=2)
