"""Argument checks of the 8-bit cache's C entries (rejected before anything touches a GPU), its oracle
against PyTorch's own 8-bit type, and the sizes of its workspace."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import kv_cache as oracle
from talm_amd import _lib
from talm_amd.kv_cache import CacheLayer

PTR = 1 << 12  # a fake address: never dereferenced on rejection


def _status(name, *args):
    lib = _lib.lib()
    status = getattr(lib, name)(*args)
    return status, lib.talm_last_error().decode()


def _write(**bad):
    v = dict(k=PTR, ks=256, v=PTR, vs=256, rows=4, kv=2, d=128, dtype=_lib.TALM_F16, bounds=PTR, past=PTR, seqs=2,
             new=1, codes=PTR, scales=PTR, tail=PTR, table=PTR, pages=8, width=4, cos=PTR, sin=PTR, cs=128, q=PTR,
             qs=1536, nq=12, out=PTR)
    v.update(bad)
    return _status("talm_cache_write", v["k"], v["ks"], 128, v["v"], v["vs"], 128, v["rows"], v["kv"], v["d"],
                   v["dtype"], v["bounds"], v["past"], v["seqs"], v["new"], v["codes"], v["scales"], v["tail"],
                   v["table"], v["pages"], v["width"], v["cos"], v["sin"], v["cs"], v["q"], v["qs"], 128, v["nq"],
                   v["out"], None)


@pytest.mark.parametrize("bad,word", [
    ({"d": 96}, "shape"), ({"dtype": _lib.TALM_F32}, "shape"), ({"kv": 0}, "shape"), ({"kv": 2000}, "shape"),
    ({"rows": -1}, "shape"), ({"rows": 1 << 31}, "shape"), ({"pages": 1 << 31}, "shape"), ({"width": -1}, "shape"),
    ({"width": (1 << 24) + 1}, "shape"), ({"new": -1}, "shape"), ({"nq": -1}, "shape"), ({"seqs": -1}, "shape"),
    ({"seqs": (1 << 24) + 1}, "shape"),
    ({"sin": None}, "cos"), ({"cos": None, "sin": None}, "cos"), ({"cs": 64}, "cos"), ({"cs": 130}, "cos"),
    ({"k": None}, "null"), ({"tail": None}, "null"), ({"codes": None}, "null"), ({"out": None}, "null"), ({"past": None}, "null"),
    ({"ks": 129}, "strides"), ({"qs": 4}, "strides"), ({"vs": -256}, "strides"), ({"k": PTR + 2}, "16-byte"),
    ({"out": PTR + 8}, "16-byte"), ({"cos": PTR + 4}, "16-byte"),
    ({"seqs": 1 << 20, "kv": 1024, "rows": 1 << 30, "new": 64}, "too many")])
def test_write_rejects(bad, word):
    status, message = _write(**bad)
    assert status == _lib.TALM_EINVAL and word in message, message


def test_calls_of_nothing_launch_nothing():
    assert _write(rows=0, k=None)[0] == _lib.TALM_OK
    assert _write(seqs=0, nq=0)[0] == _lib.TALM_OK
    assert _write(new=0, nq=0)[0] == _lib.TALM_OK
    assert _write(width=0, nq=0, codes=None, pages=0)[0] == _lib.TALM_OK
    for more in ({"rows": 0}, {"seqs": 0}, {"new": 0}, {"len": 0}, {"width": 0}):
        assert _attn(**more)[0] == _lib.TALM_OK
    for more in ({"rows": 0}, {"seqs": 0}, {"new": 0}, {"width": 0}):
        assert _read(**more)[0] == _lib.TALM_OK


def _read(**bad):
    v = dict(codes=PTR, length=PTR, seqs=2, kv=2, d=64, dtype=_lib.TALM_BF16, new=1, rows=4, k=PTR, v=PTR, width=4)
    v.update(bad)
    return _status("talm_cache_read", v["codes"], PTR, PTR, PTR, 8, v["width"], v["seqs"], v["kv"], v["d"], v["dtype"],
                   v["length"], PTR, PTR, v["new"], v["rows"], v["k"], v["v"], None)


@pytest.mark.parametrize("bad,word", [
    ({"d": 32}, "shape"), ({"dtype": 7}, "shape"), ({"rows": -1}, "shape"), ({"new": -1}, "shape"),
    ({"length": None}, "null"), ({"k": None}, "null"), ({"codes": PTR + 1}, "16-byte"), ({"v": PTR + 4}, "16-byte"),
    ({"seqs": 1 << 20, "kv": 1024, "rows": 1 << 30, "new": 64}, "too many")])
def test_read_rejects(bad, word):
    status, message = _read(**bad)
    assert status == _lib.TALM_EINVAL and word in message, message


def _attn(**bad):
    v = dict(q=PTR, qs=1536, rows=2, nq=12, kv=2, d=128, dtype=_lib.TALM_F16, bounds=PTR, seqs=2, new=1, len=9000,
             tail=PTR, pages=8, width=400, scale=0.1, window=0, sinks=0, out=PTR, ws=PTR, bytes=1 << 30)
    v.update(bad)
    return _status("talm_cache_attn", v["q"], v["qs"], 128, v["rows"], v["nq"], v["kv"], v["d"], v["dtype"],
                   v["bounds"], PTR, v["seqs"], v["new"], v["len"], PTR, PTR, v["tail"], PTR, v["pages"], v["width"],
                   v["scale"], v["window"], v["sinks"], v["out"], v["ws"], v["bytes"], None)


@pytest.mark.parametrize("bad,word", [
    ({"nq": 5}, "shape"), ({"nq": 0}, "shape"), ({"kv": 0}, "shape"), ({"d": 256}, "shape"), ({"new": -1}, "shape"),
    ({"len": -1}, "shape"), ({"len": (1 << 30) + 1}, "shape"), ({"window": -1}, "shape"), ({"sinks": -1}, "shape"),
    ({"rows": 1 << 31}, "shape"), ({"dtype": _lib.TALM_F32}, "shape"), ({"scale": 0.0}, "scale"),
    ({"scale": -1.0}, "scale"), ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"),
    ({"q": None}, "null"), ({"out": None}, "null"), ({"tail": None}, "null"), ({"qs": 4}, "strides"),
    ({"q": PTR + 8}, "16-byte"), ({"ws": PTR + 4}, "16-byte"), ({"bytes": 100}, "workspace"),
    ({"ws": None, "bytes": 0}, "workspace"), ({"ws": None}, "workspace"),
    ({"rows": 70000, "seqs": 65536, "len": 64}, "sequences")])
def test_attention_rejects(bad, word):
    status, message = _attn(**bad)
    assert status == _lib.TALM_EINVAL and word in message, message


def test_workspace_is_what_the_parts_need():
    size = _lib.lib().talm_cache_attn_workspace
    for bad in ((2, 5, 2, 128, 2, 1, 100, 0, 0), (2, 12, 2, 96, 2, 1, 100, 0, 0), (-1, 12, 2, 128, 2, 1, 100, 0, 0)):
        assert size(*bad) == -1
    # a row's keys within one part: none
    assert size(2, 12, 2, 128, 2, 1, 64, 0, 0) == 0
    parts = size(1, 12, 2, 128, 1, 1, 131072, 0, 0) // (12 * 130 * 4)
    assert 2 <= parts <= 256 and size(1, 12, 2, 128, 1, 1, 131072, 0, 0) == parts * 12 * 130 * 4
    # a window's keys, not the whole length's; windows and sinks past every length are no larger
    assert 0 < size(1, 12, 2, 128, 1, 1, 131072, 4096, 4) < size(1, 12, 2, 128, 1, 1, 131072, 0, 0)
    assert size(1, 12, 2, 128, 1, 1, 9000, 2 ** 31 - 1, 2 ** 31 - 1) == size(1, 12, 2, 128, 1, 1, 9000, 0, 0)
    # many sequences: bounded, and so are the workgroups (8192 over the KV heads)
    for rows in (64, 1000, 20000):
        assert size(rows, 64, 8, 128, rows, 1, 131072, 0, 0) <= 1 << 27
    assert size(2000, 12, 2, 128, 2000, 1, 131072, 0, 0) == 2000 * 12 * 2 * 130 * 4
    # counts of new tokens past the rows mean the rows
    assert size(1, 12, 2, 128, 1, 1 << 20, 9000, 0, 0) == size(1, 12, 2, 128, 1, 1, 9000, 0, 0)


def test_oracle_rounds_as_the_type():
    x = torch.randn(1 << 14, generator=torch.Generator().manual_seed(0)) * 60
    x = torch.cat((x, x * 2.0 ** -12, torch.tensor([448.0, -448.0, 0.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -6])))
    want = x.to(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(oracle.nearest_code(x.double().numpy()), want)


def test_oracle_scales_are_the_smallest_that_hold_the_block():
    for top, scale in ((448.0, 1.0), (449.0, 2.0), (224.0, 0.5), (224.5, 1.0), (65504.0, 256.0), (1.0, 2.0 ** -8),
                       (0.0, 1.0), (2.0 ** -24, 2.0 ** -32), (2.0 ** -133, 2.0 ** -100)):
        assert oracle.block_scale(np.array([[0.0, -top, np.inf, np.nan]])) == scale, top


def test_oracle_orders_are_permutations():
    for d in (64, 128):
        x = np.arange(64 * d).reshape(64, d)
        for order in (oracle.key_order, oracle.value_order):
            assert sorted(order(x)) == list(range(64 * d))


def test_layers_of_what_is_not_held():
    for bad in ((1, 2, 96, 64), (1, 2, 128, -1), (-1, 2, 128, 64)):
        with pytest.raises(ValueError):
            CacheLayer.allocate(*bad, device="cpu")
    with pytest.raises(ValueError):
        CacheLayer.allocate(1, 2, 128, 64, torch.float32, "cpu")
    layer = CacheLayer.allocate(3, 2, 64, 65, torch.bfloat16, "cpu")
    assert layer.capacity == 128 and layer.codes.shape == (6, 2, 2, 4096) and layer.table.tolist()[1] == [2, 3]


def test_cpu_buffers_are_refused():
    layer = CacheLayer.allocate(1, 2, 64, 64, device="cpu")
    x = torch.zeros(1, 2, 1, 64, dtype=torch.float16)
    one, bounds = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)
    for call in (lambda: layer.write(x, x, bounds, one, 1), lambda: layer.attention(x, bounds, one, 1, 1, 1.0),
                 lambda: layer.read(one, bounds, one, 1, 1)):
        with pytest.raises(ValueError, match="cache"):
            call()
    with pytest.raises(ValueError, match="window"):
        layer.attention(x, bounds, one, 1, 1, 1.0, window=0)


def test_signatures_are_bound():
    assert _lib.SIGNATURES["talm_cache_attn"][19] is ctypes.c_float
