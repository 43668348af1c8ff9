"""Calls over 8-bit rows without a GPU."""
import pytest

import kv_offload_proto_b200 as kp


def test_the_layer_step_before_init_raises():
    with pytest.raises(RuntimeError, match="kvops not inited"):
        kp.kvops().sieve_import_quant(*([0] * 17), [0], 0, 0, "e4m3", "fp16", 512, 64, 0, 0, 1, 0)
    for bad in (dict(row_format="fp8"), dict(row_dtype="fp32")):
        args = dict(row_format="e4m3", row_dtype="fp16")
        args.update(bad)
        with pytest.raises(ValueError, match="row_"):
            kp.kvops().sieve_import_quant(*([0] * 17), [0], 0, 0, args["row_format"], args["row_dtype"], 512, 64, 0, 0, 1, 0)
