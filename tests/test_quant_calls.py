"""Calls over 8-bit rows without a GPU."""
import pytest
import torch

import kv_offload_proto_b200 as kp
from kv_offload_proto_b200 import pool as pool_module
from kv_offload_proto_b200.pool import DevicePool


def test_the_layer_step_before_init_raises():
    with pytest.raises(RuntimeError, match="kvops not inited"):
        kp.kvops().sieve_import_quant(*([0] * 17), [0], 0, 0, "e4m3", "fp16", 512, 64, 0, 0, 1, 0)
    for bad in (dict(row_format="fp8"), dict(row_dtype="fp32")):
        args = dict(row_format="e4m3", row_dtype="fp16")
        args.update(bad)
        with pytest.raises(ValueError, match="row_"):
            kp.kvops().sieve_import_quant(*([0] * 17), [0], 0, 0, args["row_format"], args["row_dtype"], 512, 64, 0, 0, 1, 0)


class Launches:
    """In the place of the launch module: counts what a pool launches."""

    def __init__(self):
        self.names = []

    def __getattr__(self, name):
        if name == "quant_row_bytes":
            return kp.kvops().quant_row_bytes
        if name == "alloc_status":
            return lambda n: 0
        return lambda *args, **named: self.names.append(name)


class Batch:
    """The tensors of a coordinator that a layer-step passes on."""

    top_k, device_buffer_size, padded_buffer_size, visited_stride_b, max_num_reqs, pool_size = 4, 16, 16, 64, 2, 2

    def __getattr__(self, name):
        return torch.zeros((1, 2, 16), dtype=torch.int32)


def pool_of(monkeypatch, row_format, **kw):
    k = Launches()
    monkeypatch.setattr(pool_module, "_kvops_module", lambda: k)
    return DevicePool(0, 1, 32, 1152, segment_addrs=[1 << 20], row_format=row_format, **kw), k


def calls_of(pool, rows):
    t = torch.zeros((2, 4), dtype=torch.int32)
    return {
        "write_all": lambda: pool.batch_write_alllayers(0, 1, rows, 0),
        "write": lambda: pool.batch_write(0, t, t, t, t, t, t, rows, 2, 4),
        "read": lambda: pool.batch_read(0, t, t, t, t, t, t, rows, 2, 4),
        "step": lambda: pool.sieve_and_read(Batch(), 0, t, rows),
    }


HALF, BF, F32, BYTES, WORDS = (torch.zeros(4, dtype=d) for d in (torch.float16, torch.bfloat16, torch.float32, torch.uint8,
                                                                 torch.int32))


@pytest.mark.parametrize("call", ["write_all", "write", "read", "step"])
@pytest.mark.parametrize("kw, good, bad", [
    (dict(row_format="e4m3"), [HALF, BYTES, WORDS, 1 << 20], [BF, F32]),
    (dict(row_format="int8", row_dtype=torch.bfloat16), [BF, BYTES, WORDS, 1 << 20], [HALF, F32]),
    (dict(row_format="e4m3", hot_quantized=True), [BYTES, WORDS, 1 << 20], [HALF, BF, F32]),
    (dict(row_format="raw"), [HALF, BF, F32, BYTES, WORDS, 1 << 20], []),
])
def test_rows_of_another_type_are_refused(monkeypatch, call, kw, good, bad):
    pool, k = pool_of(monkeypatch, **kw)
    if kw.get("hot_quantized") and call == "write_all":  # whose rows are 16-bit ones all the same
        good, bad = [HALF] + good, [BF, F32]
    for rows in good:
        before = len(k.names)
        calls_of(pool, rows)[call]()
        assert len(k.names) == before + 1
    for rows in bad:
        before, cursor = len(k.names), pool._status_cursor
        with pytest.raises(ValueError, match="this pool's"):
            calls_of(pool, rows)[call]()
        assert len(k.names) == before and pool._status_cursor == cursor
