"""The paged decoder step (cruise_decoder_step_paged) at its edges: refusals of
the C entry before anything is launched, rows it leaves out, wide tables, large
batches, tables and logits in other forms, other streams."""

from __future__ import annotations

import pytest
import torch

from scenario import rel_err_rows
from test_gpu_decoder_step_paged import GEOMETRY, TOL, _pair, _tables

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


# ---- what a decode loop does with the step ---------------------------------------------------


def batch(rows, width, seed, used=4):
    """Rows of up to ``used`` blocks each, in tables ``width`` blocks wide."""
    gen = torch.Generator().manual_seed(seed)
    shape = (GEOMETRY["num_layers"], rows * used, BLOCK, GEOMETRY["num_kv_heads"], GEOMETRY["head_dim"])
    key, value = (torch.randn(shape, generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
    table = torch.full((rows, width), -1, dtype=torch.int32)
    table[:, :used] = torch.randperm(rows * used, generator=gen).int().reshape(rows, used)
    token = torch.randint(0, GEOMETRY["vocab"], (rows,), generator=gen)
    position = torch.randint(0, used * BLOCK, (rows,), generator=gen)
    return token.cuda(), position.cuda(), table.cuda(), key, value


def close(a, b):
    assert float(rel_err_rows(a.float().cpu().flatten(1), b.float().cpu().flatten(1)).max()) <= TOL


def workspace(engine, rows, width):
    return engine.lib.cruise_decoder_attention_workspace(rows, GEOMETRY["num_heads"], GEOMETRY["num_kv_heads"],
                                                         GEOMETRY["head_dim"], width * BLOCK, 0)


def test_wide_tables_take_the_split_form(engine):
    """Tables for 32000 positions: the engine's attention is split over all CTAs and
    joined, with a workspace of the engine's that later calls share."""
    assert workspace(engine, 4, 4) == 0 and workspace(engine, 4, 2000) == workspace(engine, 64, 4000) > 0
    for rows, width in ((4, 2000), (64, 4000), (3, 2000), (4, 2000)):
        token, position, table, key, value = batch(rows, width, seed=rows)
        narrow_key, narrow_value = key.clone(), value.clone()
        narrow = engine.decoder_step_paged(token, position, table[:, :4].contiguous(), narrow_key, narrow_value)
        wide = engine.decoder_step_paged(token, position, table, key, value)
        close(wide, narrow)
        for a, b in ((key, narrow_key), (value, narrow_value)):
            close(a.flatten(0, 3), b.flatten(0, 3))


@pytest.mark.parametrize("rows", [129, 200, 256])
def test_batches_past_one_token_tile(engine, rows):
    token, position, table, key, value = batch(rows, 4, seed=rows)
    k1, v1 = key.clone(), value.clone()
    together = engine.decoder_step_paged(token, position, table, key, value)
    for r in (0, rows // 2, rows - 1):
        one = engine.decoder_step_paged(token[r:r + 1], position[r:r + 1], table[r:r + 1], k1, v1)
        close(one, together[r:r + 1])


def test_fp32_tables_of_the_same_values_give_the_same_step(engine):
    token, position, table, key, value = batch(5, 4, seed=80)
    cos, sin = _tables(engine, BLOCK * 4)
    assert cos.dtype == torch.bfloat16
    k1, v1 = key.clone(), value.clone()
    want = engine.decoder_step_paged(token, position, table, k1, v1, cos, sin)
    got = engine.decoder_step_paged(token, position, table, key, value, cos.float(), sin.float())
    assert torch.equal(got, want) and torch.equal(key, k1) and torch.equal(value, v1)


def test_logits_inside_a_wider_tensor(engine):
    token, position, table, key, value = batch(5, 4, seed=81)
    want = engine.decoder_step_paged(token, position, table, key.clone(), value.clone())
    room = torch.full((5, GEOMETRY["vocab"] + 24), 7.0, dtype=torch.bfloat16, device="cuda")
    got = engine.decoder_step_paged(token, position, table, key, value, logits_out=room[:, 8:-16])
    assert got.data_ptr() == room[:, 8:].data_ptr() and torch.equal(got, want)
    assert (room[:, :8] == 7).all() and (room[:, -16:] == 7).all()


def test_the_step_follows_the_current_stream(engine):
    """Inputs written late on another stream, and a reader on it right after."""
    token, position, table, key, value = batch(6, 4, seed=82)
    k1, v1 = key.clone(), value.clone()
    want = engine.decoder_step_paged(token, position, table, k1, v1)
    late = [torch.zeros_like(token), torch.full_like(position, -1), torch.zeros_like(key)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        for to, source in zip(late, (token, position, key)):
            to.copy_(source)
        got = engine.decoder_step_paged(late[0], late[1], table, late[2], value).clone()
    stream.synchronize()
    assert torch.equal(got, want) and torch.equal(late[2], k1) and torch.equal(value, v1)
