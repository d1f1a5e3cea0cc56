"""The paged decoder step (cruise_decoder_step_paged) at its edges: refusals of
the C entry before anything is launched."""

from __future__ import annotations

import pytest
import torch

from test_gpu_decoder_step_paged import GEOMETRY, _pair

pytestmark = pytest.mark.gpu

BLOCK, WIDTH = 16, 4


@pytest.fixture(scope="module")
def engine():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    engine, _, _ = _pair(GEOMETRY, BLOCK, WIDTH)
    yield engine
    torch.cuda.synchronize()
    engine.close()


def tensors(rows=4, blocks=16):
    shape = (GEOMETRY["num_layers"], blocks, BLOCK, GEOMETRY["num_kv_heads"], GEOMETRY["head_dim"])
    cuda = dict(device="cuda")
    return dict(token=torch.arange(rows, **cuda), position=torch.arange(rows, **cuda),
                key=torch.zeros(shape, dtype=torch.bfloat16, **cuda), value=torch.zeros(shape, dtype=torch.bfloat16, **cuda),
                table=torch.arange(rows * WIDTH, dtype=torch.int32, **cuda).view(rows, WIDTH),
                cos=torch.ones(BLOCK * WIDTH, 128, **cuda), sin=torch.zeros(BLOCK * WIDTH, 128, **cuda),
                logits=torch.zeros(rows, GEOMETRY["vocab"], dtype=torch.bfloat16, **cuda))


def step(engine, t, **change):
    """The C call on the tensors' addresses, or on those in ``change``."""
    at = {name: x.data_ptr() for name, x in t.items()}
    at.update(change)
    rows, blocks = t["token"].shape[0], t["key"].shape[1]
    rc = engine.lib.cruise_decoder_step_paged(
        engine.handle, rows, at["token"], at["position"], at["key"], at["value"], blocks, BLOCK, at["table"], WIDTH, WIDTH,
        at["cos"], at["sin"], 2, BLOCK * WIDTH, at["logits"], GEOMETRY["vocab"], torch.cuda.current_stream().cuda_stream)
    why = engine.lib.cruise_epoch_last_error(engine.handle)
    return rc, why.decode() if why else ""


@pytest.mark.parametrize("name", ["cos", "sin", "token", "position", "key", "value", "table", "logits"])
def test_host_memory_is_refused(engine, name):
    t = tensors()
    host = t[name].cpu()
    for there in (host, host.pin_memory()):
        rc, why = step(engine, t, **{name: there.data_ptr()})
        assert rc == -1 and ("device memory" in why or "aligned" in why), (rc, why)
    assert not t["key"].any() and not t["logits"].any()


@pytest.mark.parametrize("name", ["token", "position", "key", "value", "table", "logits"])
def test_missing_arrays_are_refused(engine, name):
    rc, why = step(engine, tensors(), **{name: None})
    assert rc == -1 and "NULL" in why, (rc, why)


@pytest.mark.parametrize("name, off", [("cos", 8), ("sin", 4), ("key", 8), ("value", 2), ("token", 4), ("position", 4),
                                       ("table", 2), ("logits", 1)])
def test_unaligned_arrays_are_refused(engine, name, off):
    t = tensors()
    rc, why = step(engine, t, **{name: t[name].data_ptr() + off})
    assert rc == -1 and "aligned" in why, (rc, why)
    assert not t["key"].any() and not t["logits"].any()


@pytest.mark.parametrize("name, other, off", [
    ("value", "key", 0), ("value", "key", 4096), ("key", "value", 64), ("logits", "key", 0), ("logits", "value", 65536),
    ("token", "key", 128), ("position", "value", 8), ("table", "key", 4), ("cos", "key", 256), ("sin", "value", 0),
    ("logits", "token", 0), ("logits", "position", 16), ("logits", "table", 4), ("cos", "logits", 512), ("sin", "logits", 0),
])
def test_overlapping_arrays_are_refused(engine, name, other, off):
    t = tensors()
    rc, why = step(engine, t, **{name: t[other].data_ptr() + off})
    assert rc == -1 and "overlap" in why, (rc, why)
    assert not t["key"].any() and not t["logits"].any()


def test_arrays_side_by_side_are_taken(engine):
    t = tensors()
    want = {name: x.clone() for name, x in t.items()}
    assert step(engine, want)[0] == 0
    both = torch.zeros(2, *t["key"].shape, dtype=torch.bfloat16, device="cuda")
    t.update(key=both[0], value=both[1])
    rc, why = step(engine, t)
    assert rc == 0, why
    assert torch.equal(t["logits"], want["logits"]) and torch.equal(t["key"], want["key"]) and torch.equal(t["value"], want["value"])


def rows_left_out(engine, **change):
    """The step with a row 2 that has to be left out against the step without it."""
    t = tensors()
    want = {name: x.clone() for name, x in t.items()}
    want["position"][2] = -1
    assert step(engine, want)[0] == 0
    for name, value in change.items():
        t[name] = value(t[name])
    rc, why = step(engine, t)
    assert torch.equal(t["key"], want["key"]) and torch.equal(t["value"], want["value"])
    others = [0, 1, 3]
    assert torch.equal(t["logits"][others], want["logits"][others])
    return rc, why


@pytest.mark.parametrize("entry", [-1, 16, 2 ** 31 - 1, -2 ** 31])
def test_a_position_without_a_block_is_an_error(engine, entry):
    def spoil(table):
        table[2, 0] = entry
        return table

    rc, why = rows_left_out(engine, table=spoil)
    assert rc == -5 and "row 2" in why and "block" in why, (rc, why)


def test_a_position_past_the_rotation_tables_is_an_error(engine):
    from cruise_b200.engine import EngineError

    t = tensors()
    t["position"][2] = 40
    t["cos"], t["sin"] = t["cos"][:40], t["sin"][:40]
    want = {name: x.clone() for name, x in t.items()}
    want["position"][2] = -1
    call = lambda t, **keep: engine.decoder_step_paged(t["token"], t["position"], t["table"], t["key"], t["value"], **keep)  # noqa: E731
    logits = call(want, cos=want["cos"], sin=want["sin"])
    with pytest.raises(EngineError, match=r"\(-5\).*row 2.*rotation tables \(40 rows\)"):
        call(t, cos=t["cos"], sin=t["sin"], logits_out=t["logits"])
    assert torch.equal(t["key"], want["key"]) and torch.equal(t["value"], want["value"])
    assert torch.equal(t["logits"][[0, 1, 3]], logits[[0, 1, 3]])
    # the engine's own tables end where its resident rows do
    t = tensors(rows=2, blocks=24)
    t["table"] = torch.arange(24, dtype=torch.int32, device="cuda").view(2, 12)
    t["position"][:] = torch.tensor([127, 128])
    with pytest.raises(EngineError, match=r"row 1.*\(128 rows\)"):
        call(t)
    t["position"][1] = 126
    call(t)


def test_rows_that_do_not_exist_stay_inactive(engine):
    t = tensors()
    t["token"][0], t["token"][1] = -1, GEOMETRY["vocab"]
    t["position"][2], t["position"][3] = -5, BLOCK * WIDTH
    t["table"][:] = -1
    rc, why = step(engine, t)
    assert rc == 0, why
    assert not t["key"].any() and not t["value"].any()


def test_the_same_arrays_are_taken(engine):
    t = tensors()
    rc, why = step(engine, t)
    assert rc == 0, why
    assert t["logits"].any() and t["key"].any()
