"""The decoder step over caller-held paged caches (cruise_decoder_step_paged) and
the host loop under logit rules, on the GPU.

* One step against the oracle's decoder step on the same caches and inputs, at
  contexts past what a resident row holds, with an inactive row: logits within
  2e-2 per row and the new K/V within 2e-2 per head vector (the bound of the
  resident step's test), everything else in the caches untouched.
* The paged step against the resident step on the same caches.
* A greedy decode loop of the paged step and ``choose`` keeps the oracle's tokens.
* The host loop under rules equals the same loop with the rules applied on the
  host, and without rules the plain one.
"""

from __future__ import annotations

from dataclasses import replace

import numpy as np
import pytest
import torch

from cruise_b200.host_loop import HostLoopError, RuledChoice, host_loop_epoch
from decoder_reference import choose_reference
from oracle.decoder import OracleDecoder
from oracle.model import OracleConfig, seeded_weights
from scenario import decode_inputs, make_scenario, prefill_epochs, rel_err_rows

pytestmark = pytest.mark.gpu

TOL = 2e-2
GEOMETRY = dict(num_layers=2, hidden=512, num_heads=4, num_kv_heads=1, head_dim=128, intermediate=1024, vocab=4096)
ODD = dict(num_layers=1, hidden=448, num_heads=7, num_kv_heads=1, head_dim=64, intermediate=688, vocab=4096)


def _pair(geometry, block_size, blocks_per_row, seed=0):
    """An engine whose own rows hold 2 blocks, and an oracle over a longer cache."""
    from cruise_b200.engine import EpochEngine
    from cruise_b200.model_config import ModelConfig

    engine = EpochEngine(ModelConfig(name="paged", block_size=64, blocks_per_row=2, num_blocks=8, configured_eos=4095, **geometry))
    engine.init_synthetic(seed)
    ocfg = OracleConfig(block_size=block_size, blocks_per_row=blocks_per_row, num_blocks=4 * blocks_per_row, **geometry)
    return engine, ocfg, OracleDecoder(ocfg, seeded_weights(ocfg, seed=seed))


def _tables(engine, capacity):
    from cruise_b200.engine import rope_tables

    config = engine.config
    cos, sin = rope_tables(replace(config, block_size=capacity, blocks_per_row=1))
    return cos.cuda(), sin.cuda()


def _caches(ocfg, seed):
    gen = torch.Generator().manual_seed(seed)
    shape = (ocfg.num_layers, ocfg.num_blocks, ocfg.block_size, ocfg.num_kv_heads, ocfg.head_dim)
    return [torch.randn(shape, generator=gen).to(torch.bfloat16) for _ in range(2)], gen


@pytest.mark.parametrize("geometry, block_size, blocks_per_row, positions", [
    (GEOMETRY, 16, 100, [1599, 0, 777, 63]),
    (GEOMETRY, 128, 2, [200, 127, 128, 5]),
    (ODD, 24, 30, [700, 1, 23, 24]),
])
def test_paged_step_matches_the_oracle_step(cuda_ok, geometry, block_size, blocks_per_row, positions):
    engine, ocfg, oracle = _pair(geometry, block_size, blocks_per_row)
    (key, value), gen = _caches(ocfg, 3)
    table = torch.randperm(ocfg.num_blocks, generator=gen).to(torch.int32).reshape(4, blocks_per_row)
    token = torch.randint(0, ocfg.vocab, (4,), generator=gen)
    position = torch.tensor(positions)
    active = torch.tensor([1, 1, 1, 0], dtype=torch.int32)
    slot = table[torch.arange(4), position // block_size] * block_size + position % block_size
    want, want_key, want_value, _ = oracle.step(token, position, (position + 1).int(), table, slot.int(), key, value, active)
    cos, sin = _tables(engine, block_size * blocks_per_row)
    gk, gv = key.cuda(), value.cuda()
    given = torch.where(active.bool(), position, -1)
    logits = engine.decoder_step_paged(token.cuda(), given.cuda(), table.cuda(), gk, gv, cos, sin)
    err = rel_err_rows(logits[:3].float().cpu(), want[:3])
    assert float(err.max()) <= TOL, f"logits rel err {float(err.max()):.3g}"
    flat = lambda c: c.cpu().reshape(ocfg.num_layers, -1, ocfg.num_kv_heads, ocfg.head_dim)  # noqa: E731
    for got, wanted, before in ((gk, want_key, key), (gv, want_value, value)):
        got, wanted, before = flat(got), flat(wanted), flat(before)
        new = slot[:3].long()
        a, b = got[:, new].float(), wanted[:, new].float()
        rel = (a - b).norm(dim=-1) / b.norm(dim=-1).clamp_min(1e-6)
        assert float(rel.max()) <= TOL
        rest = torch.ones(got.shape[1], dtype=torch.bool)
        rest[new] = False
        assert torch.equal(got[:, rest], before[:, rest])
    engine.close()


@pytest.mark.parametrize("geometry", ["tiny", "7b-2l"])
def test_paged_step_agrees_with_the_resident_step(cuda_ok, geometry):
    """The same caches, tables and inputs through both steps."""
    from cruise_b200.engine import EpochEngine
    from cruise_b200.model_config import QWEN25_7B, TINY

    cfg = TINY if geometry == "tiny" else replace(QWEN25_7B, name="qwen2.5-7b-2l", num_layers=2)
    engine = EpochEngine(cfg)
    engine.init_synthetic(0)
    sc = make_scenario(vocab=cfg.vocab, seed=9, token_high=min(cfg.vocab, 151643))
    for inputs in prefill_epochs(sc, cfg.block_size, cfg.vocab):
        assert engine.run(**inputs).status == 0
    inputs = decode_inputs(sc, cfg.block_size)
    rows = [r for r in range(4) if inputs["active"][r]]
    caches = [c.cuda() for c in engine.read_kv()]
    want, _ = engine.decoder_step(inputs["token"], inputs["position"], inputs["seq_len"], inputs["slot"], inputs["active"],
                                  inputs["block_table"])
    position = torch.from_numpy(np.where(inputs["active"] != 0, inputs["position"], -1)).cuda()
    logits = engine.decoder_step_paged(torch.from_numpy(inputs["token"]).cuda(), position,
                                       torch.from_numpy(inputs["block_table"]).reshape(4, -1).int().cuda(), *caches)
    err = rel_err_rows(logits[rows].float().cpu(), torch.from_numpy(want[rows]))
    assert float(err.max()) <= TOL
    engine.close()


def test_paged_step_of_many_rows(cuda_ok):
    """37 rows with a full table each equal the same rows taken one by one, up to
    the order of fp32 sums (the projections tile by row count)."""
    engine, ocfg, _ = _pair(GEOMETRY, 16, 40)
    rows, gen = 37, torch.Generator().manual_seed(4)
    shape = (ocfg.num_layers, rows * 4, 16, ocfg.num_kv_heads, ocfg.head_dim)
    key, value = (torch.randn(shape, generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
    table = torch.randperm(rows * 4, generator=gen).int().reshape(rows, 4).cuda()
    token = torch.randint(0, ocfg.vocab, (rows,), generator=gen).cuda()
    position = torch.randint(0, 64, (rows,), generator=gen).cuda()
    k1, v1 = key.clone(), value.clone()
    together = engine.decoder_step_paged(token, position, table, key, value)
    for r in (0, 5, 36):
        one = engine.decoder_step_paged(token[r:r + 1], position[r:r + 1], table[r:r + 1], k1, v1)
        assert float(rel_err_rows(one.float().cpu(), together[r:r + 1].float().cpu()).max()) <= TOL
    assert torch.equal(engine.decoder_step_paged(token, position, table, key, value), together)   # same bits again
    engine.close()


def test_paged_greedy_loop_keeps_the_oracle_tokens(cuda_ok):
    """Decode from empty caches: the paged step and choose on the device; every
    token is the oracle's, or within the oracle's near ties (top-2 margin 2e-2)."""
    from cruise_b200.decoder_ops import choose

    engine, ocfg, oracle = _pair(GEOMETRY, 16, 12)
    shape = (ocfg.num_layers, ocfg.num_blocks, 16, ocfg.num_kv_heads, ocfg.head_dim)
    key, value = (torch.zeros(shape, dtype=torch.bfloat16) for _ in range(2))
    gk, gv = key.cuda(), value.cuda()
    table = torch.arange(ocfg.num_blocks, dtype=torch.int32).reshape(4, -1)
    cos, sin = _tables(engine, 16 * 12)
    token = torch.tensor([11, 200, 3000, 4000])
    position = torch.zeros(4, dtype=torch.int64)
    for _ in range(40):
        slot = (table[torch.arange(4), position // 16] * 16 + position % 16).int()
        want, key, value, _ = oracle.step(token, position, (position + 1).int(), table, slot, key, value, torch.ones(4, dtype=torch.int32))
        logits = engine.decoder_step_paged(token.cuda(), position.cuda(), table.cuda(), gk, gv, cos, sin)
        chosen = choose(logits).cpu()
        best = want.max(dim=1).values
        margin = best - want[torch.arange(4), chosen]
        assert float((margin / best.abs().clamp_min(1e-3)).max()) <= 2e-2
        token, position = chosen, position + 1
    engine.close()


def test_paged_step_refuses(cuda_ok):
    from cruise_b200.engine import EngineError

    engine, ocfg, _ = _pair(GEOMETRY, 16, 4)
    shape = (ocfg.num_layers, 16, 16, ocfg.num_kv_heads, ocfg.head_dim)
    args = dict(token=torch.zeros(4, dtype=torch.int64, device="cuda"), position=torch.zeros(4, dtype=torch.int64, device="cuda"),
                block_table=torch.arange(16, dtype=torch.int32, device="cuda").view(4, 4),
                key=torch.zeros(shape, dtype=torch.bfloat16, device="cuda"), value=torch.zeros(shape, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError, match="token must be"):
        engine.decoder_step_paged(**{**args, "token": args["token"].int()})
    with pytest.raises(ValueError, match="on cuda"):
        engine.decoder_step_paged(**{**args, "position": args["position"].cpu()})
    with pytest.raises(ValueError, match="value must be"):
        engine.decoder_step_paged(**{**args, "value": args["value"][:, :8]})
    with pytest.raises(ValueError, match="both rotation"):
        engine.decoder_step_paged(**args, cos=torch.zeros(8, 128, device="cuda"))
    many = 4 * 64 + 1
    with pytest.raises(EngineError, match="rows outside"):
        engine.decoder_step_paged(torch.zeros(many, dtype=torch.int64, device="cuda"), torch.zeros(many, dtype=torch.int64, device="cuda"),
                                  torch.zeros(many, 1, dtype=torch.int32, device="cuda"), args["key"], args["value"])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(EngineError, match="captured"):
        with torch.cuda.graph(graph):
            engine.decoder_step_paged(**args)
    # rows that do not exist are inactive: nothing is stored
    before = args["key"].clone()
    args.update(token=torch.tensor([-1, 4096, 5, 6], device="cuda"), position=torch.tensor([0, 0, -3, 64], device="cuda"))
    engine.decoder_step_paged(**args)
    assert torch.equal(args["key"], before) and not args["value"].any()
    engine.close()


# ---- the host loop under logit rules -------------------------------------------------------

def _loop(engine, sc, inputs, choose=None, device_logits=True):
    cfg = engine.config
    for prefill in prefill_epochs(sc, cfg.block_size, cfg.vocab):
        assert engine.run(**prefill).status == 0
    room = torch.empty(4, cfg.vocab, device="cuda") if device_logits else None
    return host_loop_epoch(lambda *a: engine.decoder_step(*a, logits_out=room), inputs, cfg.block_size, cfg.capacity, choose=choose)


def _tiny_engine():
    from cruise_b200.engine import EpochEngine

    engine = EpochEngine("tiny")
    engine.init_synthetic(0)
    return engine


def test_host_loop_without_effective_rules_is_the_plain_loop(cuda_ok):
    plain, ruled = _tiny_engine(), _tiny_engine()
    vocab = plain.config.vocab
    sc = make_scenario(vocab=vocab, seed=12, k=8)
    inputs = decode_inputs(sc, plain.config.block_size)
    want = _loop(plain, sc, inputs, device_logits=False)
    got = _loop(ruled, sc, inputs, RuledChoice(vocab, [[1, 2], [3], [], [4]], 64))
    np.testing.assert_array_equal(got[0], want[0])
    np.testing.assert_array_equal(got[1], want[1])
    plain.close()
    ruled.close()


class HostRules:
    """RuledChoice's definition on the host: choose_reference on copies."""

    def __init__(self, device: RuledChoice):
        self.history = device.history.cpu().clone()
        self.prompt, self.length = device.prompt_len.cpu(), device.history_len.cpu().clone()
        self.rules = {k: v.cpu() for k, v in device.rules.items()}
        self.allowed = None if device.allowed is None else device.allowed.cpu()

    def __call__(self, logits, active):
        flags = torch.as_tensor(np.asarray(active, dtype=np.int32))
        _, token = choose_reference(torch.as_tensor(logits).cpu(), self.history, self.prompt, self.length, **self.rules,
                                    allowed=self.allowed, active=flags, dtype=torch.float32)
        for r in range(4):
            if token[r] >= 0:
                self.history[r, self.length[r]] = token[r]
                self.length[r] += 1
        return token.numpy()


def test_host_loop_under_rules_equals_the_rules_on_the_host(cuda_ok):
    device, host = _tiny_engine(), _tiny_engine()
    vocab = device.config.vocab
    sc = make_scenario(vocab=vocab, seed=13, k=8)
    inputs = decode_inputs(sc, device.config.block_size)
    gen = torch.Generator().manual_seed(1)
    allowed = torch.randint(-2 ** 31, 2 ** 31, (4, vocab // 32), generator=gen).int()
    allowed[0] = -1
    rules = RuledChoice(vocab, [[5, 6, 7]] * 4, 64, repetition=[1.5, 1.2, 1.0, 2.0], frequency=0.4, presence=[0.3, 0.0, 0.1, 0.0],
                        bias=[{17: 3.0, 5: -1.0}, None, {}, {4000: 2.5}], allowed=allowed.cuda())
    reference = HostRules(rules)
    got = _loop(device, sc, inputs, rules)
    want = _loop(host, sc, inputs, reference, device_logits=False)
    np.testing.assert_array_equal(got[0], want[0])
    np.testing.assert_array_equal(got[1], want[1])
    assert torch.equal(rules.history_len.cpu(), reference.length)
    assert torch.equal(rules.history.cpu(), reference.history)
    bits = allowed.numpy().view(np.uint32)
    for step in got[0]:
        for r, token in enumerate(step):
            if token >= 0:
                assert (bits[r, token // 32] >> (token % 32)) & 1
    device.close()
    host.close()


def test_host_loop_fails_where_no_token_is_left(cuda_ok):
    engine = _tiny_engine()
    vocab = engine.config.vocab
    sc = make_scenario(vocab=vocab, seed=14)
    rules = RuledChoice(vocab, [[]] * 4, 8, allowed=torch.zeros(4, vocab // 32, dtype=torch.int32, device="cuda"))
    with pytest.raises(HostLoopError) as err:
        _loop(engine, sc, decode_inputs(sc, engine.config.block_size), rules)
    assert err.value.code == 23
    engine.close()


def test_ruled_choice_refuses(cuda_ok):
    with pytest.raises(ValueError, match="does not fit"):
        RuledChoice(10, [[1, 2, 3]], 2)
    with pytest.raises(ValueError, match="values"):
        RuledChoice(10, [[1]], 2, frequency=[0.1, 0.2])
    with pytest.raises(ValueError, match="bias lists"):
        RuledChoice(10, [[1]], 2, bias=[None, None])
