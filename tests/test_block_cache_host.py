"""What the block cache and the rotary positions refuse, and their host arithmetic: no GPU needed."""
import ctypes
import math

import pytest
import torch

from nanokv_b200 import _lib, ops
from nanokv_b200.block_cache import BlockCache
from nanokv_b200.rotary import Rotary, frequencies


def struct(*, lengths=(10, 20), kv_heads=2, head_dim=128, blocks=4, dtype=_lib.NKV_BF16, address=256):
    array = (ctypes.c_int32 * len(lengths))(*lengths)
    return _lib.BlockCache(address, address, address, address, address, address, array, len(lengths), kv_heads, head_dim, blocks, dtype)


def rows(heads, address=256):
    return _lib.Tokens(address, 1024, 512, 128, heads)


def status_of(name, *args):
    lib = _lib.library()
    return getattr(lib, name)(*args), lib.nkv_last_error().decode()


@pytest.mark.parametrize("change,word", [
    (dict(head_dim=96), "head width"), (dict(dtype=_lib.NKV_F32), "bf16 or fp16"), (dict(blocks=0), "blocks"),
    (dict(kv_heads=0), "kv_heads"), (dict(lengths=(10, 257)), "257 tokens"), (dict(lengths=(-1,)), "tokens"),
    (dict(address=264), "aligned"), (dict(address=0), "missing")])
def test_caches_that_are_refused(change, word):
    for name, args in (("nkv_block_append", (rows(2), rows(2), 1, None, None, None)), ("nkv_block_read", (0, 1, 256, 256, None)),
                       ("nkv_block_attend", (rows(2), 1, None, 1, 1.0, 256, 256, None, 256, None, 0, None))):
        status, text = status_of(name, struct(**change), *args)
        assert status in (_lib.NKV_ERR_INVALID, _lib.NKV_ERR_UNSUPPORTED) and word in text, (name, text)


def test_calls_that_are_refused():
    counts = (ctypes.c_int32 * 2)(1, 5)
    for name, args, word in (
            ("nkv_block_append", (struct(), rows(2), rows(2), 240, None, None, None), "do not fit"),
            ("nkv_block_append", (struct(), rows(1), rows(2), 1, None, None, None), "heads"),
            ("nkv_block_append", (struct(), rows(2), rows(2), 4, counts, None, None), "5 of 4"),
            ("nkv_block_append", (struct(), rows(2), rows(2), -1, None, None, None), "tokens"),
            ("nkv_block_append", (struct(), rows(2, address=None), rows(2), 1, None, None, None), "no rows"),
            ("nkv_block_append", (struct(), rows(2), rows(2), 1, None, _lib.Rotation(256, 256, 8, 24, 0), None), "multiple of 16"),
            ("nkv_block_append", (struct(), rows(2), rows(2), 1, None, _lib.Rotation(256, 256, 8, 256, 0), None), "rotary_dim"),
            ("nkv_block_read", (struct(), 3, 2, 256, 256, None), "tokens 3 to 2"),
            ("nkv_block_read", (struct(), 0, 257, 256, 256, None), "tokens 0 to 257"),
            ("nkv_block_read", (struct(), 0, 1, 256, 264, None), "aligned"),
            ("nkv_block_attend", (struct(), rows(3), 1, None, 1, 1.0, 256, 256, None, 256, None, 0, None), "3 query heads"),
            ("nkv_block_attend", (struct(), rows(2), 4, counts, 1, 1.0, 256, 256, None, 256, None, 0, None), "5 of 4"),
            ("nkv_block_attend", (struct(), rows(2), 1, None, 1, 1.0, 256, None, None, 256, None, 0, None), "missing"),
            ("nkv_block_attend", (struct(), rows(2), 1, None, 1, 1.0, 256, 256, 256, 256, None, 0, None), "workspace"),
            ("nkv_block_evict", (256, 256, counts, counts, 2, 1, 8, 2, 1, 2, 512, 512, None), "to keep"),
            ("nkv_block_evict", (256, 256, counts, counts, 2, 1, 8, 4, 1, 2, 256, 512, None), "in place"),
            ("nkv_block_evict", (256, 256, counts, counts, 2, 1, 8, 4, 1, 2, 512, 512, None), "open blocks"),
            ("nkv_rotary", (rows(2), 256, None, None, _lib.NKV_BF16, 1, 1, 64, _lib.Rotation(256, 256, 8, 66, 0), 0, None), "rotary_dim"),
            ("nkv_rotary", (rows(2), 256, None, None, _lib.NKV_BF16, 1, 1, 64, _lib.Rotation(256, 256, 8, 31, 0), 0, None), "rotary_dim"),
            ("nkv_rotary", (rows(2), 256, None, None, _lib.NKV_BF16, 1, 1, 64, _lib.Rotation(256, 256, 8, 32, 2), 0, None), "layout"),
            ("nkv_rotary", (rows(2), 256, None, None, _lib.NKV_BF16, 1, 1, 64, _lib.Rotation(None, 256, 8, 32, 0), 0, None), "arrays"),
            ("nkv_rotary", (rows(2), 256, None, None, 7, 1, 1, 64, _lib.Rotation(256, 256, 8, 32, 0), 0, None), "dtype")):
        status, text = status_of(name, *args)
        assert status in (_lib.NKV_ERR_INVALID, _lib.NKV_ERR_TOO_LARGE) and word in text, (name, text)
        with pytest.raises(ValueError):
            _lib.check(status)


def test_calls_without_work_do_nothing():
    assert status_of("nkv_block_append", struct(), rows(2), rows(2), 0, None, None, None)[0] == 0
    assert status_of("nkv_block_read", struct(), 5, 5, None, None, None)[0] == 0
    assert status_of("nkv_rotary", rows(2), None, None, None, _lib.NKV_BF16, 1, 0, 64, _lib.Rotation(256, 256, 8, 32, 0), 0, None)[0] == 0
    assert status_of("nkv_block_evict", None, None, None, None, 0, 1, 8, 4, 1, 2, None, None, None)[0] == 0


def test_there_is_no_cpu_path():
    x = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16)
    positions = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        Rotary(64, 8, device="cpu").apply(x, positions=positions)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        BlockCache(1, 1, 64, 64, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.block_evict(torch.zeros(1, 1, 4), torch.zeros(1, 1, 4, dtype=torch.int32), [4], [0], keep=2)


def test_arrays_that_make_no_cache():
    def arrays(**change):
        made = dict(k_codes=torch.zeros(1, 2, 3, 64, 128, dtype=torch.uint8), v_codes=torch.zeros(1, 2, 3, 128, 64, dtype=torch.uint8),
                    scales=torch.zeros(1, 2, 3, 2), table=torch.zeros(1, 2, 3, dtype=torch.int32),
                    k_tail=torch.zeros(1, 2, 64, 128, dtype=torch.bfloat16), v_tail=torch.zeros(1, 2, 128, 64, dtype=torch.bfloat16),
                    lengths=[0])
        made.update(change)
        return BlockCache.over(*made.values())
    for change, word in ((dict(scales=torch.zeros(1, 2, 3)), "scales"), (dict(table=torch.zeros(1, 2, 3)), "table"),
                         (dict(v_codes=torch.zeros(1, 2, 3, 64, 128, dtype=torch.uint8)), "v_codes"),
                         (dict(k_tail=torch.zeros(1, 2, 64, 128)), "bf16 or fp16"),
                         (dict(v_tail=torch.zeros(1, 2, 128, 64, dtype=torch.float16)), "v_tail"),
                         (dict(k_codes=torch.zeros(1, 2, 3, 64, 96, dtype=torch.uint8)), "64 or 128"),
                         (dict(k_codes=torch.zeros(1, 2, 3, 32, 128, dtype=torch.uint8)), "k_codes")):
        with pytest.raises(ValueError, match=word):
            arrays(**change)
    with pytest.raises(ValueError, match="positive"):
        BlockCache(0, 1, 64, 64)


def test_frequencies():
    plain, gain = frequencies(8, base=100.0)
    assert gain == 1.0 and torch.allclose(plain, 100.0 ** -(torch.arange(4).double() / 4), rtol=1e-14)
    linear, _ = frequencies(8, base=100.0, scaling=dict(kind="linear", factor=4.0))
    assert torch.allclose(linear, plain / 4, rtol=1e-14)
    base, _ = frequencies(8, base=100.0, scaling=dict(kind="base", factor=4.0))
    assert math.isclose(float(base[0]), 1.0) and math.isclose(float(base[-1]), float(plain[-1]) / 4, rel_tol=1e-12)
    blend, gain = frequencies(64, scaling=dict(kind="blend", factor=8.0, trained=4096))
    plain, _ = frequencies(64)
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(blend[turns >= 32], plain[turns >= 32]) and torch.allclose(blend[turns <= 1], plain[turns <= 1] / 8, rtol=1e-14)
    between = (turns > 1) & (turns < 32)
    assert between.any() and (blend < plain)[between].all() and (blend > plain / 8)[between].all()
    assert math.isclose(gain, 0.1 * math.log(8) + 1)
    for bad in (dict(kind="other", factor=2.0), dict(kind="linear", factor=0.5), dict(kind="blend", factor=2.0, trained=64, low=4.0, high=4.0)):
        with pytest.raises(ValueError):
            frequencies(8, scaling=bad)
    for dim in (0, 3, -2):
        with pytest.raises(ValueError):
            frequencies(dim)


def test_rotary_tables_that_are_refused():
    for table, kw, word in ((torch.zeros(4, 8), {}, "table"), (torch.zeros(4, 40, 2), {}, "elements of heads"),
                            (torch.zeros(4, 8, 2), dict(layout="thirds"), "layout"), (torch.zeros(4, 8, 2).double(), {}, "float32")):
        with pytest.raises(ValueError, match=word):
            Rotary.over(table, head_dim=64, **kw)
