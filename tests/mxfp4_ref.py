"""The microscaled 4-bit format in 64 bits, from its definition (shared by the CPU and GPU tests)."""
import torch


def values(x: torch.Tensor) -> torch.Tensor:
    """[rows, cols] -> the float64 values its 4-bit form stands for: per 32 columns a scale 2^(floor(log2 max) - 2) within
    2^-127 .. 2^127, elements rounded half to even on steps of 1/2 (below 2), 1 (below 4) and 2, at most 6; NaN for a block
    that is not finite."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = torch.zeros(rows, blocks * 32, dtype=torch.float64, device=x.device)
    v[:, :cols] = x.double()
    v = v.view(rows, blocks, 32)
    top = v.abs().amax(2, keepdim=True)
    bad = ~torch.isfinite(v).all(2, keepdim=True)
    e = (torch.floor(torch.log2(torch.where(bad, 1.0, top))) - 2).clamp(-127, 127).long()
    scale = ((e + 1023) << 52).view(torch.float64)      # 2^e by its bits: a device's pow may be a rounding off
    y = v / scale
    step = torch.where(y.abs() >= 4, 2.0, torch.where(y.abs() >= 2, 1.0, 0.5)).to(torch.float64)
    y = (torch.round(y / step) * step).clamp(-6, 6) * scale
    return torch.where(bad, torch.nan, y).view(rows, -1)[:, :cols]
