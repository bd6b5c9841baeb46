"""per_token_cast_to_nvfp4 and its way back against the definition in 64 bits: scales and codes have to be those of the exact
quotients, on borders between two codes too."""
import pytest
import torch

from product_helpers import E2M1, e2m1_values

E4M3_POSITIVE = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def _nearest(values, levels):
    """Index of the nearest level, ties to the even index; differences from the middles are exact in 64 bits here."""
    middle = (levels[1:] + levels[:-1]) / 2
    at = torch.bucketize(values, middle)
    tie = (values == torch.cat((middle, middle[-1:] * 0 - 1))[at]) & (at % 2 == 1)
    return at + tie.long()


def _reference(x, ts):
    """(scale bytes, codes) of x (CPU) for the fp32 number ts."""
    rows, hidden = x.shape
    g = x.double().view(rows, -1, 16)
    amax = g.abs().amax(-1)
    # compare with the borders times 6 ts rather than divide: the products are exact
    scale = _nearest(amax, E4M3_POSITIVE * 6 * ts) if ts > 0 else torch.where(amax > 0, 126, 0)
    d = E4M3_POSITIVE[scale] * ts
    codes = torch.zeros_like(g, dtype=torch.int64)
    levels = torch.tensor(E2M1, dtype=torch.float64)
    for i in range(7):
        border = (levels[i] + levels[i + 1]) / 2 * d[..., None]
        codes += ((g.abs() > border) | ((g.abs() == border) & (i % 2 == 1))) & (d[..., None] > 0)
    return scale.to(torch.uint8), codes.view(rows, hidden)


def _check(x, ts, device):
    from tilekernels_b200 import quant
    scale = torch.tensor([ts], dtype=torch.float32, device=device)
    q, sf = quant.per_token_cast_to_nvfp4(x.to(device), scale)
    rows, hidden = x.shape
    assert q.dtype == torch.int8 and q.shape == (rows, hidden // 2) and q.is_contiguous()
    assert sf.dtype == torch.float8_e4m3fn and sf.shape == (rows, hidden // 16) and sf.is_contiguous()
    want_sf, want = _reference(x, scale.double().item())
    assert torch.equal(sf.cpu().view(torch.uint8), want_sf)
    u = q.cpu().view(torch.uint8).to(torch.int64)
    codes = torch.stack((u & 15, u >> 4), -1).flatten(1)
    assert torch.equal(codes & 7, want)
    signs = (codes >> 3).bool()
    assert torch.equal(signs[want > 0], (x < 0)[want > 0])
    for fmt, dtype in (('fp32', torch.float32), ('bf16', torch.bfloat16)):
        back = quant.cast_back((q, sf), fmt, (1, 16), tensor_scale=scale)
        exact = e2m1_values(q) * sf.cpu().double().repeat_interleave(16, 1) * scale.double().item()
        assert back.dtype == dtype and torch.equal(back.cpu(), exact.float().to(dtype))
    return q, sf


@pytest.mark.gpu
@pytest.mark.parametrize('rows,hidden', ((1, 16), (1, 7168), (3, 528), (257, 2048), (1000, 1040)))
@pytest.mark.parametrize('dtype', (torch.bfloat16, torch.float32), ids=('bf16', 'fp32'))
def test_codes_and_scales(cuda_device, rows, hidden, dtype):
    gen = torch.Generator().manual_seed(rows + hidden)
    x = torch.randn((rows, hidden), generator=gen)
    x[:, ::37] *= 30
    x[rows // 2] = 0
    x = x.to(dtype)
    _check(x, float(x.abs().max()) / 2688, cuda_device)


@pytest.mark.gpu
def test_quotients_on_borders(cuda_device):
    """Every border of e2m1 for every e4m3 scale, hit exactly and missed by one ulp on either side, and every border of e4m3."""
    ts = 0.0078125
    rows = []
    for s in E4M3_POSITIVE[1:].tolist():
        borders = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
        exact = torch.tensor([6.0] + borders + [-b for b in borders] + [0.5], dtype=torch.float64) * s * ts
        near = exact.float()
        rows += [near, torch.nextafter(near, near * 2), torch.nextafter(near, near * 0)]
    middles = (E4M3_POSITIVE[1:] + E4M3_POSITIVE[:-1]) / 2 * 6 * ts
    for m in middles.float():
        for v in (m, torch.nextafter(m, m * 2), torch.nextafter(m, m * 0)):
            rows.append(torch.cat((v[None], torch.linspace(0, 1, 15) * v)))
    x = torch.stack(rows)
    # the first element fixes the block's scale; one ulp off it, the scale must not move (it lies inside its interval)
    _check(x, ts, cuda_device)
    _check(x, 0.0073, cuda_device)   # a tensor scale of 24 bits: products of 28 bits
    gen = torch.Generator().manual_seed(3)
    short = torch.randint(-12, 13, (4096, 64), generator=gen).float() * 0.25   # ratios of short numbers: many exact ties
    _check(short, 3.0 / 2688, cuda_device)
    _check(short.to(torch.bfloat16), 0.25 / 6, cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize('ts', (2.0 ** -130, 2.0 ** -100, 1e-30, 1e30, 2.0 ** 120, 0.0))
def test_tensor_scales_near_the_ends(cuda_device, ts):
    gen = torch.Generator().manual_seed(9)
    x = torch.randn((64, 256), generator=gen, dtype=torch.float64)
    x = (x * (ts if ts > 0 else 1.0) * 500).clamp(-3e38, 3e38).float()
    if ts > 0 and ts < 2.0 ** -120:
        x = torch.round(x.double() / 2.0 ** -149).mul(2.0 ** -149).float()
    _check(x, ts, cuda_device)


@pytest.mark.gpu
def test_saturation_strides_and_empty(cuda_device):
    from tilekernels_b200 import quant
    ts = torch.ones(1, device=cuda_device)
    x = torch.zeros((4, 32))
    x[0, :3] = torch.tensor([float('inf'), -float('inf'), 1.0])
    x[1, 0] = 3e38
    q, sf = quant.per_token_cast_to_nvfp4(x.to(cuda_device), ts)
    assert torch.equal(sf.cpu().float(), torch.tensor([[448.0, 0], [448.0, 0], [0, 0], [0, 0]]))
    assert e2m1_values(q)[0, :3].tolist() == [6.0, -6.0, 0.0] and e2m1_values(q)[1, 0] == 6.0
    gen = torch.Generator().manual_seed(5)
    wide = torch.randn((33, 512), generator=gen).to(torch.bfloat16).to(cuda_device)
    for view in (wide[:, 8:264], wide[::2, :128], wide[1:, 16:32]):   # rows on 16- and 32-byte boundaries
        got, want = quant.per_token_cast_to_nvfp4(view, ts * 0.01), quant.per_token_cast_to_nvfp4(view.contiguous(), ts * 0.01)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1].view(torch.uint8), want[1].view(torch.uint8))
    q, sf = quant.per_token_cast_to_nvfp4(wide[:0], ts)
    assert q.shape == (0, 256) and sf.shape == (0, 32)
    assert quant.cast_back((q, sf), 'bf16', (1, 16), tensor_scale=ts).shape == (0, 512)


@pytest.mark.gpu
def test_refusals(cuda_device):
    from tilekernels_b200 import quant
    ts = torch.ones(1, device=cuda_device)
    x = torch.zeros((4, 64), device=cuda_device)
    for bad in (x[:, :24], x.half(), x.T, x[0]):
        with pytest.raises(AssertionError):
            quant.per_token_cast_to_nvfp4(bad, ts)
    with pytest.raises(AssertionError):
        quant.per_token_cast_to_nvfp4(x, 1.0)
    with pytest.raises(AssertionError):
        quant.per_token_cast_to_nvfp4(x, ts.double())
    with pytest.raises(AssertionError):
        quant.per_token_cast_to_nvfp4(x, ts.cpu())
    with pytest.raises(RuntimeError, match='16-byte'):
        quant.per_token_cast_to_nvfp4(torch.zeros((4, 66), device=cuda_device)[:, 1:33], ts)
    q, sf = quant.per_token_cast_to_nvfp4(x, ts)
    with pytest.raises(AssertionError):
        quant.cast_back((q, sf), 'bf16', (1, 16))
    with pytest.raises(AssertionError):
        quant.cast_back((q, sf), 'bf16', (1, 32), tensor_scale=ts)
    with pytest.raises(AssertionError):
        quant.cast_back(quant.per_token_cast(x, 'e2m1', 32), 'bf16', (1, 32), tensor_scale=ts)


def test_cpu_tensors_are_refused():
    from tilekernels_b200 import quant
    with pytest.raises(AssertionError):
        quant.per_token_cast_to_nvfp4(torch.zeros((4, 64)), torch.ones(1))


@pytest.mark.parametrize('rows,blocks', ((5, 1), (1, 1), (4, 3)))
def test_other_casts_refuse_e4m3_scales(rows, blocks):
    """One block per row, or transposed scales: unit stride along rows, which float32 and packed scales have in column-major
    storage.  Read as float32, e4m3 bytes would be read four times as far as they reach."""
    from tilekernels_b200 import quant
    from tilekernels_b200.quant.common import get_cast_input_and_config
    data = torch.zeros((rows, blocks * 8), dtype=torch.int8)
    sf = torch.zeros((blocks, rows), dtype=torch.uint8).view(torch.float8_e4m3fn).T
    assert sf.stride(0) == 1
    for block in ((1, 16), (1, 32)):
        with pytest.raises(AssertionError, match='scales'):
            get_cast_input_and_config((data, sf), block)
    with pytest.raises(AssertionError, match='scales'):
        quant.per_token_cast((data, sf), 'e4m3', 16, (1, 16))
    with pytest.raises(AssertionError, match='scales'):
        quant.per_block_cast_lossless((data, sf), 'e4m3', (1, 16), (1, 32))
    for dtype in (torch.bfloat16, torch.uint8):
        with pytest.raises(AssertionError, match='scales'):
            get_cast_input_and_config((data, torch.zeros((blocks, rows), dtype=dtype).T), (1, 32))
