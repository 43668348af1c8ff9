"""The decode driver's checks of stored rows and its refusals, on the CPU."""
import numpy as np
import pytest
import torch

import quant_model
from kv_offload_proto_b200.decode import FINITE, attention_error, main, parse_args, row_matches


def test_new_options_default_to_what_ran_before():
    a = parse_args([])
    assert a.row_format == "raw" and a.attend_heads == 0 and a.draft_tokens == 1


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_a_row_matches_what_its_codes_stand_for_and_no_other(fmt):
    rng = np.random.default_rng(1)
    words = rng.integers(0, 2 ** 32, 288, dtype=np.uint32) & np.uint32(FINITE)
    row = words.view(np.float16)
    assert np.isfinite(row).all() and np.abs(row).max() < 2
    stored = quant_model.encode(torch.from_numpy(row[None].copy()), fmt, 512)
    back = quant_model.decode(stored, fmt, "fp16", 512)[0].numpy()
    assert row_matches(back, row, fmt, 512)
    assert not row_matches(back, row, "raw", 512) and row_matches(row, row, "raw", 512)
    for at, by in ((5, 0.3), (400, -0.3), (570, 2.0 ** -10)):
        wrong = back.copy()
        wrong[at] += np.float16(by)
        assert not row_matches(wrong, row, fmt, 512), at


def test_attention_error_tells_right_from_wrong():
    g = torch.Generator().manual_seed(2)
    q, keys, drafts = (torch.randn(s, generator=g).half() for s in ((2, 3, 576), (20, 576), (2, 576)))
    out, lse = torch.empty((2, 3, 512), dtype=torch.float16), torch.empty((2, 3))
    for t in range(2):
        k = torch.cat([keys, drafts[:t + 1]]).double()
        s = q[t].double() @ k.T * 576 ** -0.5
        out[t], lse[t] = (torch.softmax(s, 1) @ k[:, :512]).half(), torch.logsumexp(s, 1).float()
    assert attention_error(torch, q, keys, 576 ** -0.5, drafts, out, lse) <= 1
    assert attention_error(torch, q, keys, 576 ** -0.5, None, out, lse) > 1
    assert attention_error(torch, q, keys[:-1], 576 ** -0.5, drafts, out, lse) > 1


@pytest.mark.parametrize("extra", [
    ["--attend-heads", "8", "--shared-hot"], ["--attend-heads", "129"], ["--attend-heads", "8", "--draft-tokens", "65"],
    ["--attend-heads", "8", "--kv-lora-rank", "256"], ["--row-format", "int8", "--kv-lora-rank", "500", "--qk-rope", "12"],
])
def test_refusals(tmp_path, extra, capsys):
    assert main(["--run-dir", str(tmp_path), *extra]) == 1
    assert "[xds][ERROR]" in capsys.readouterr().out
