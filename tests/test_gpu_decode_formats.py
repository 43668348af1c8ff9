"""The decode driver over pools that store rows in 8 bits and with each step's attention: every step's rows, SIEVE
outputs and first request's attention are checked by the driver itself, in a fresh process each."""
import re

import pytest

from test_gpu_decode_driver import run_driver

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("extra", [
    ("--attend-heads", "8"),
    ("--row-format", "e4m3", "--attend-heads", "16", "--draft-tokens", "4", "--steps", "6"),
    ("--row-format", "int8", "--attend-heads", "128", "--segment-devices", "0,-1,0", "--stripe-rows", "2", "--injective",
     "--one-call", "--layer-rows", "4096"),
    ("--row-format", "e4m3", "--kv-lora-rank", "128", "--qk-rope", "0"),
])
def test_driver_with_stored_rows_and_attention(tmp_path, extra):
    rc, out = run_driver(tmp_path, "--layer-rows", "2048", "--oracle", *extra)
    assert rc == 0, out[-3000:]
    assert "[xds][ERROR]" not in out and "[xds] all done" in out
    steps = re.findall(r"\[xds\] step \d+: layer=\d+ miss=(\d+) rows in [\d.]+ us \(checked=(\d+)\)", out)
    assert len(steps) >= 6 and all(int(m) > 0 and int(c) > 0 for m, c in steps)
    attended = re.findall(r"\[xds\] step \d+: attended \d+ tokens x \d+ heads of 8 requests", out)
    assert len(attended) == (len(steps) if "--attend-heads" in extra else 0)
