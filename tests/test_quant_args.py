"""The 8-bit row codec and the attention's arguments, without a GPU: sizes, refusals, the codec
model itself against its formula in 64 bits, and the tree's words."""
import numpy as np
import pytest
import torch

import kv_offload_proto_b200 as kp
import quant_model
from kv_offload_proto_b200.offload import XdsOffloadCoordinator, tree_masks
from kv_offload_proto_b200.pool import dtype_name


def test_stored_row_sizes():
    mod = kp.kvops()
    assert mod.quant_row_bytes("e4m3", "fp16") == 656
    for quant, plain in ((128, 0), (256, 64), (512, 64), (640, 8), (4096, 4096)):
        for fmt in ("e4m3", "int8"):
            n = mod.quant_row_bytes(fmt, "bf16", quant, plain)
            assert n == quant_model.stored_bytes(quant, plain) and n % 16 == 0


@pytest.mark.parametrize("args, message", [
    (("raw", "fp16", 512, 64), "row_format"),
    (("e5m2", "fp16", 512, 64), "row_format"),
    (("int8", "fp32", 512, 64), "row_dtype"),
    (("int8", "fp16", 0, 64), "quant_elems"),
    (("int8", "fp16", 500, 64), "quant_elems"),
    (("int8", "fp16", 4224, 64), "quant_elems"),
    (("int8", "fp16", 512, 60), "plain_elems"),
    (("int8", "fp16", 512, 4104), "plain_elems"),
])
def test_codec_refusals(args, message):
    with pytest.raises((RuntimeError, ValueError), match=message):
        kp.kvops().quant_row_bytes(*args)


def test_calls_before_init_raise():
    mod = kp.kvops()
    with pytest.raises(RuntimeError, match="kvops not inited"):
        mod.export_quant_alllayer([0], 0, "e4m3", "fp16", 512, 64, *([0] * 7))
    with pytest.raises(RuntimeError, match="kvops not inited"):
        mod.export_quant([0], 0, 0, "e4m3", "fp16", 512, 64, *([0] * 11))
    with pytest.raises(RuntimeError, match="kvops not inited"):
        mod.import_quant([0], 0, 0, "e4m3", "fp16", 512, 64, *([0] * 11))
    with pytest.raises(RuntimeError, match="kvops not inited"):
        mod.attend_workspace(1, 1, 1, 1, 0)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_codec_model_is_within_half_a_step(fmt, dtype):
    """What a row reads back as is off by at most half a step of its code (e4m3: 2^-4 of the
    value, or half of the smallest code 2^-9; int8: half of 1) in units of the scale, and half a
    step of the 16-bit type; the fp32 operations on the way (three, each off by 2^-24 of the value)
    may add 2^-22 of the largest code and carry a value across the middle between two codes."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn((40, 576), generator=g)
    x *= torch.exp(torch.randn((40, 576), generator=g) * 2)
    rows = x.to(quant_model.TORCH[dtype])
    back = quant_model.decode(quant_model.encode(rows, fmt, 512), fmt, dtype, 512)
    assert torch.equal(back[:, 512:], rows[:, 512:])
    v = rows[:, :512].double().numpy().reshape(40, 4, 128)
    got = back[:, :512].double().numpy().reshape(40, 4, 128)
    unit = np.abs(v).max(-1, keepdims=True) / float(quant_model.TOP[fmt])
    half = np.maximum(np.abs(v) * 2.0 ** -4, unit * 2.0 ** -10) if fmt == "e4m3" else unit * 0.5
    eps = torch.finfo(quant_model.TORCH[dtype]).eps / 2
    tiny = torch.finfo(quant_model.TORCH[dtype]).smallest_normal * eps
    assert (np.abs(got - v) <= half + eps * (np.abs(v) + half) + unit * 448 * 2.0 ** -22 + tiny).all()


def test_codec_model_of_odd_groups():
    rows = torch.zeros((4, 512), dtype=torch.bfloat16)
    rows[0, 5] = float("inf")
    rows[1, 200] = float("nan")
    rows[2, 300] = 1e-33  # below 2^-100: stored as zeros
    rows[3, 400] = -3.0
    for fmt in ("e4m3", "int8"):
        back = quant_model.decode(quant_model.encode(rows, fmt, 512), fmt, "bf16", 512).float()
        assert back[0, :128].isnan().all() and (back[0, 128:] == 0).all()
        assert back[1, 128:256].isnan().all() and (back[1, :128] == 0).all()
        assert (back[2] == 0).all()
        assert back[3, 400] == -3.0 and (back[3, :384] == 0).all()


def test_tree_masks():
    m = tree_masks([[-1, 0, 0, 1, 3, -1]])
    assert m.tolist() == [[1, 3, 5, 11, 27, 32]]
    chain = tree_masks(torch.arange(64) - 1)
    assert chain[63].item() == -1 and chain[62].item() == 2 ** 63 - 1
    for bad in ([0], [-1, 1], [-2], [-1] * 65):
        with pytest.raises(ValueError):
            tree_masks(bad)
    with pytest.raises(ValueError):
        tree_masks(torch.zeros(2))


def test_dtype_names():
    assert dtype_name(torch.float16) == "fp16" and dtype_name("bf16") == "bf16"
    for bad in (torch.float32, "fp8", None):
        with pytest.raises(ValueError):
            dtype_name(bad)


class HostCoordinator(XdsOffloadCoordinator):
    _require_cuda = False


def coordinator(reqs=2, k=8):
    co = HostCoordinator("cpu", 1, reqs, 16, k, reqs, 64)
    co._req_pool_indices = torch.arange(reqs)
    return co


HOT = torch.zeros(2 * 16 * 576, dtype=torch.float16)
Q = torch.zeros((2, 4, 576), dtype=torch.float16)


@pytest.mark.parametrize("change, message", [
    (dict(q=torch.zeros((2, 4, 512), dtype=torch.float16)), "q must be"),
    (dict(q=torch.zeros((2, 4, 576))), "float16 or bfloat16"),
    (dict(q=torch.zeros((2, 4, 1152), dtype=torch.float16)[..., ::2]), "unit last stride"),
    (dict(q=torch.zeros((3, 4, 576), dtype=torch.float16)), "batch rows"),
    (dict(topk_device_slots=torch.zeros((2, 8), dtype=torch.int64)), "topk_device_slots"),
    (dict(topk_device_slots=torch.zeros((1, 8), dtype=torch.int32)), "topk_device_slots"),
    (dict(topk_device_slots=torch.zeros((2, 3, 8), dtype=torch.int32)), "topk_device_slots"),
    (dict(topk_device_slots=torch.zeros((2, 16), dtype=torch.int32)[:, ::2]), "topk_device_slots"),
    (dict(row_format="fp8"), "row_format"),
    (dict(draft_rows=torch.zeros((2, 1, 512), dtype=torch.float16)), "draft_rows"),
    (dict(draft_rows=torch.zeros((2, 1, 576), dtype=torch.bfloat16)), "draft_rows"),
    (dict(draft_rows=torch.zeros((1, 1, 576), dtype=torch.float16)), "draft_rows"),
    (dict(tree=torch.zeros((2, 1), dtype=torch.int32)), "tree"),
    (dict(tree=torch.zeros((2, 2), dtype=torch.int64)), "tree"),
    (dict(hot_row_base=HOT[:-1]), "hot rows must"),
    (dict(hot_rows=17), "hot rows must"),
    (dict(out=torch.zeros((2, 4, 512))), "out"),
    (dict(out=torch.zeros((2, 4, 511), dtype=torch.float16)), "out"),
    (dict(lse=torch.zeros((2, 4), dtype=torch.float16)), "lse"),
])
def test_attend_refusals(change, message):
    args = dict(q=Q, hot_row_base=HOT, hot_req_stride_rows=16)
    args.update(change)
    with pytest.raises(ValueError, match=message):
        coordinator().attend(args.pop("q"), args.pop("hot_row_base"), **args)


def test_attend_needs_a_batch():
    co = HostCoordinator("cpu", 1, 2, 16, 8, 2, 64)
    with pytest.raises(RuntimeError, match="set_batch"):
        co.attend(Q, HOT, hot_req_stride_rows=16)
    with pytest.raises(RuntimeError, match="kvops not inited"):
        coordinator().attend(Q, HOT, hot_req_stride_rows=16)


def test_null_outputs_are_refused_at_the_c_entries():
    import ctypes
    import os

    import kv_offload_proto_b200 as kp

    kp.install_kvops_ext()
    lib = ctypes.CDLL(os.path.join(os.path.dirname(kp.__file__), "libkvops_b200.so"))
    lib.kvops_last_error.restype = ctypes.c_char_p
    assert lib.kvops_quant_row_bytes(1, 0, 512, 64, None) != 0
    assert b"NULL" in lib.kvops_last_error()
    size = ctypes.c_uint32()
    assert lib.kvops_quant_row_bytes(1, 0, 512, 64, ctypes.byref(size)) == 0 and size.value == 656
