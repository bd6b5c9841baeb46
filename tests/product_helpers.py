"""Plain forms in 64 bits of the matrix products, quantized operands for them, and error bounds by arithmetic.

A sum of k fp32 terms formed in any order, each addition cutting off at most one unit in the last place (2^-23 of the
partial sum, which is at most the sum of magnitudes S), is off by at most k * 2^-23 * S.  Rounding to bf16 adds at most
half a step, 2^-8 of the result."""
import torch

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def e2m1_values(q: torch.Tensor) -> torch.Tensor:
    u = q.cpu().view(torch.uint8).to(torch.int64)
    codes = torch.stack((u & 15, u >> 4), dim=-1).flatten(-2)
    v = torch.tensor(E2M1, dtype=torch.float64)[codes & 7]
    return torch.where(codes >= 8, -v, v)


def dequantized(q: torch.Tensor, sf: torch.Tensor, block) -> torch.Tensor:
    """(rows, k) in 64 bits; sf int32 words of four exponent bytes, or float8_e4m3fn."""
    v = e2m1_values(q) if q.dtype == torch.int8 else q.cpu().to(torch.float64)
    rows, k = v.shape
    r, c = torch.arange(rows) // block[0], torch.arange(k) // block[1]
    sf = sf.cpu()
    if sf.dtype == torch.float8_e4m3fn:
        return v * sf.to(torch.float64)[r][:, c]
    byte = (sf.to(torch.int64)[r][:, c // 4] >> (8 * (c % 4))) & 255
    return v * torch.exp2((byte - 127).double())


def assert_product(got: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0) -> None:
    """got = scale * a @ b.T, a and b in 64 bits."""
    want = scale * (a @ b.T)
    k = a.shape[1]
    bound = k * 2.0 ** -23 * abs(scale) * (a.abs() @ b.abs().T)
    if got.dtype == torch.bfloat16:
        bound = bound + 2.0 ** -8 * (want.abs() + bound)
    off = (got.cpu().double() - want).abs()
    assert torch.isfinite(got.float()).all()
    worst = (off - bound).max().item() if off.numel() else 0.0
    assert worst <= 0, f'off by {worst:.3e} more than the bound; relative error {off.norm() / want.norm():.3e}'


def segments(sizes, align=1, first=0, gap=0):
    """Starts and ends of groups of these sizes, and the row behind the last one."""
    start, end, at = [], [], first
    for n in sizes:
        at = -(-at // align) * align
        start.append(at)
        end.append(at + n)
        at += n + gap
    return start, end, at


def int32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)
