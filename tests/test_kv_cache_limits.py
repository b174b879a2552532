"""Calls of the 8-bit cache's C entries that are larger than a launch, refused before anything touches a GPU: an
axis of a launch has fewer than 2^32 threads, 2^24 workgroups of 256."""

import pytest
import torch

from talm_amd import _lib
from test_kv_cache_args import _attn, _read, _write


@pytest.mark.parametrize("bad", [
    # a tile of 64 rows each: 2^24 of them, one too many
    {"rows": 1 << 30, "nq": 1, "kv": 1, "seqs": 2, "new": 1 << 29, "len": 1 << 20, "width": 1 << 14},
    {"rows": 1 << 30, "nq": 8, "kv": 4, "seqs": 1, "new": (1 << 29) - 1, "len": 64, "d": 64, "qs": 512}])
def test_attention_of_more_tiles_than_a_launch(bad):
    status, message = _attn(**bad)
    assert status == _lib.TALM_EINVAL and "too many" in message, message


@pytest.mark.skipif(torch.cuda.is_available(), reason="launches on fake addresses where there is a GPU")
def test_writes_and_reads_of_more_workgroups_than_a_launch_are_taken():
    """512 sequences of 8 heads, any of which may have a prompt of 131072 rows: launched in parts (here without a
    device, so the error is the launch's and no refusal)."""
    many = {"seqs": 512, "kv": 8, "d": 64, "rows": 140000, "new": 131072, "width": 4096}
    for call, more in ((_write, {"nq": 0, "ks": 512, "vs": 512, "cs": 64}), (_read, {})):
        status, message = call(**many, **more)
        assert status == _lib.TALM_EHIP, message
