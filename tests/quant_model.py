"""The 8-bit row codec in numpy, one IEEE fp32 operation at a time, for the tests."""
import numpy as np
import torch

GROUP = 128
TOP = {"e4m3": np.float32(448), "int8": np.float32(127)}
TORCH = {"fp16": torch.float16, "bf16": torch.bfloat16}


def scale_bytes(quant):
    return (quant // GROUP * 4 + 15) // 16 * 16


def stored_bytes(quant, plain):
    return quant + scale_bytes(quant) + 2 * plain


def encode(rows, fmt, quant):
    """[n, quant + plain] torch 16-bit rows (CPU) -> [n, stored] uint8 numpy."""
    n, plain = rows.shape[0], rows.shape[1] - quant
    x = rows[:, :quant].float().numpy().reshape(n, quant // GROUP, GROUP)
    with np.errstate(all="ignore"):
        a = np.abs(x).max(-1)  # numpy's max gives NaN where there is one
        bad, none = ~np.isfinite(a), a < np.float32(2.0 ** -100)
        safe = np.where(bad | none, np.float32(1), a)
        inv = (TOP[fmt] / safe).astype(np.float32)
        y = (np.where((bad | none)[..., None], np.float32(0), x) * inv[..., None]).astype(np.float32)
        scale = np.where(bad, np.float32(np.nan), np.where(none, np.float32(0), (safe / TOP[fmt]).astype(np.float32)))
    y = y.reshape(n, quant)
    if fmt == "e4m3":
        codes = torch.from_numpy(y).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    else:
        codes = np.rint(y).astype(np.int8).view(np.uint8)
    out = np.zeros((n, stored_bytes(quant, plain)), np.uint8)
    out[:, :quant] = codes
    out[:, quant:quant + quant // GROUP * 4] = scale.astype(np.float32).view(np.uint8).reshape(n, -1)
    out[:, quant + scale_bytes(quant):] = rows[:, quant:].contiguous().view(torch.uint8).numpy().reshape(n, -1)
    return out


def decode(stored, fmt, dtype, quant):
    """[n, stored] uint8 numpy -> [n, quant + plain] torch 16-bit rows."""
    n = stored.shape[0]
    c = torch.from_numpy(np.ascontiguousarray(stored[:, :quant]))
    c = (c.view(torch.float8_e4m3fn).float() if fmt == "e4m3" else c.view(torch.int8).float()).numpy()
    s = np.ascontiguousarray(stored[:, quant:quant + quant // GROUP * 4]).view(np.float32)
    with np.errstate(all="ignore"):
        x = (c.reshape(n, -1, GROUP) * s[..., None]).astype(np.float32).reshape(n, quant)
    plain = torch.from_numpy(np.ascontiguousarray(stored[:, quant + scale_bytes(quant):])).view(TORCH[dtype])
    return torch.cat([torch.from_numpy(x).to(TORCH[dtype]), plain.reshape(n, -1)], 1)
