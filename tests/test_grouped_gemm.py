"""grouped_gemm and grouped_gemm_wgrad against products in 64 bits, group by group; rows of no group; the layer they make."""
import pytest
import torch

from product_helpers import assert_product, dequantized, int32, segments
from test_block_scaled_gemm import quantize

# group sizes: the mean decides between the tile variants, the single sizes hit their edges
SIZES = {
    'one': (1,), 'few': (1, 0, 2, 15, 16, 17, 0, 31, 33), 'skewed': (0, 0, 150, 1, 3), 'middle': (64, 127, 129, 0, 65, 63),
    'large': (257, 1, 224, 300, 0, 511), 'single': (700,),
}


def _rows(sizes, k, device, align=1, gap=0, seed=0, first=0, spare=5):
    """bf16 rows with NaN and infinities in all that belong to no group."""
    start, end, used = segments(sizes, align, first, gap)
    gen = torch.Generator().manual_seed(seed + k + sum(sizes))
    x = torch.randn((used + spare, k), generator=gen)
    member = torch.zeros(used + spare, dtype=torch.bool)
    for s, e in zip(start, end):
        member[s:e] = True
    x[~member] = float('nan')
    x[~member, ::3] = float('inf')
    return x.to(torch.bfloat16).to(device), start, end, member


def _check_groups(got, x, w, start, end, transpose=False, scale=None):
    for e, (s, t) in enumerate(zip(start, end)):
        if t > s:
            assert_product(got[s:t], x[s:t], w[e].T if transpose else w[e], 1.0 if scale is None else scale[e])


@pytest.mark.gpu
@pytest.mark.parametrize('name', SIZES)
@pytest.mark.parametrize('n,k', ((128, 64), (264, 200), (520, 1032)))
@pytest.mark.parametrize('transpose', (False, True), ids=('w', 'w_t'))
def test_bf16(cuda_device, name, n, k, transpose):
    from tilekernels_b200 import moe
    sizes = SIZES[name]
    x, start, end, member = _rows(sizes, k, cuda_device, align=4 if name == 'middle' else 1, gap=3 if name == 'large' else 0)
    gen = torch.Generator().manual_seed(n)
    w = torch.randn((len(sizes), k, n) if transpose else (len(sizes), n, k), generator=gen).to(torch.bfloat16).to(cuda_device)
    s, e = int32(start, cuda_device), int32(end, cuda_device)
    got = moe.grouped_gemm(x, w, s, e, transpose_w=transpose)
    _check_groups(got, x.cpu().double(), w.cpu().double(), start, end, transpose)
    assert (got[~member.to(cuda_device)] == 0).all()
    # into a given destination: rows of no group stay as they are
    out = torch.full((x.shape[0], n + 8), 3.0, dtype=torch.bfloat16, device=cuda_device)
    assert moe.grouped_gemm(x, w, s, e, transpose_w=transpose, out=out[:, :n]) is not None
    assert torch.equal(out[member.to(cuda_device), :n], got[member.to(cuda_device)])
    assert (out[~member.to(cuda_device)] == 3.0).all() and (out[:, n:] == 3.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize('sizes', ((1,), (20,), (0, 3), (50,), (61, 0)))
@pytest.mark.parametrize('transpose', (False, True), ids=('w', 'w_t'))
def test_few_tiles_and_a_long_k(cuda_device, sizes, transpose):
    """Products that several blocks share along k."""
    from tilekernels_b200 import moe
    n, k = 200, 3992
    x, start, end, member = _rows(sizes, k, cuda_device)
    gen = torch.Generator().manual_seed(n)
    w = torch.randn((len(sizes), k, n) if transpose else (len(sizes), n, k), generator=gen).to(torch.bfloat16).to(cuda_device)
    got = moe.grouped_gemm(x, w, int32(start, cuda_device), int32(end, cuda_device), transpose_w=transpose)
    _check_groups(got, x.cpu().double(), w.cpu().double(), start, end, transpose)
    assert (got[~member.to(cuda_device)] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize('name', SIZES)
@pytest.mark.parametrize('form', (('e4m3', (1, 128), (128, 128)), ('e4m3', (1, 32), (1, 32)), ('e2m1', (1, 32), (1, 32)),
                                  ('nvfp4', (1, 16), (1, 16))), ids=lambda f: f'{f[0]}-{f[1][1]}')
@pytest.mark.parametrize('n,k', ((128, 128), (328, 704)))
def test_quantized(cuda_device, name, form, n, k):
    from tilekernels_b200 import moe
    fmt, xb, wb = form
    sizes = SIZES[name]
    x, start, end, member = _rows(sizes, k, cuda_device, gap=1 if name == 'few' else 0)
    x[~member.to(cuda_device)] = 0
    xq, xv, xt = quantize(x, fmt, xb)
    if fmt != 'nvfp4':   # what the rows of no group hold does not matter: the largest scales and NaN codes there
        data = xq[0].clone()
        data.view(torch.uint8)[~member.to(cuda_device)] = 0x7f
        xq = (data, xq[1])
    gen = torch.Generator().manual_seed(n + k)
    parts = [quantize((torch.randn((n, k), generator=gen) * 2.0 ** (i % 5)).to(torch.bfloat16).to(cuda_device), fmt, wb) for i in range(len(sizes))]
    data = torch.stack([p[0][0].view(torch.uint8) for p in parts]).view(xq[0].dtype)
    alpha = scale = None
    if fmt == 'nvfp4':
        sf = torch.stack([p[0][1].view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn)
        alpha = xt * torch.cat([p[2] for p in parts])
        scale = alpha.double().tolist()
    else:
        sf = torch.stack([p[0][1].T.contiguous() for p in parts]).transpose(1, 2)
    got = moe.grouped_gemm(xq, (data, sf), int32(start, cuda_device), int32(end, cuda_device), xb, wb, alpha=alpha)
    _check_groups(got, xv, [p[1] for p in parts], start, end, scale=scale)
    assert (got[~member.to(cuda_device)] == 0).all()


@pytest.mark.gpu
def test_scales_of_all_experts_in_one_matrix(cuda_device):
    """The weights quantized in one call over all experts' rows."""
    from tilekernels_b200 import moe
    experts, n, k = 3, 256, 384
    x, start, end, _ = _rows((40, 0, 7), k, cuda_device, spare=0)
    gen = torch.Generator().manual_seed(1)
    w = torch.randn((experts * n, k), generator=gen).to(torch.bfloat16).to(cuda_device)
    xq, xv, _ = quantize(x, 'e4m3', (1, 128))
    for block in ((128, 128), (1, 128), (32, 32)):
        wq, wv, _ = quantize(w, 'e4m3', block)
        got = moe.grouped_gemm(xq, (wq[0].view(experts, n, k), wq[1]), int32(start, cuda_device), int32(end, cuda_device), (1, 128), block)
        _check_groups(got, xv, wv.view(experts, n, k), start, end)


@pytest.mark.gpu
@pytest.mark.parametrize('name', SIZES)
@pytest.mark.parametrize('n,k', ((8, 8), (256, 128), (264, 520), (1000, 200)))
def test_wgrad(cuda_device, name, n, k):
    from tilekernels_b200 import moe
    sizes = SIZES[name]
    x, start, end, member = _rows(sizes, k, cuda_device, gap=2, first=3)
    g, _, _, _ = _rows(sizes, n, cuda_device, gap=2, first=3, seed=1)
    s, e = int32(start, cuda_device), int32(end, cuda_device)
    for dtype in (torch.float32, torch.bfloat16):
        got = moe.grouped_gemm_wgrad(g, x, s, e, out_dtype=dtype)
        assert got.shape == (len(sizes), n, k) and got.dtype == dtype
        for i, (a, b) in enumerate(zip(start, end)):
            if a == b:
                assert (got[i] == 0).all()
            else:
                assert_product(got[i], g[a:b].cpu().double().T, x[a:b].cpu().double().T)
        assert torch.equal(moe.grouped_gemm_wgrad(g, x, s, e, out_dtype=dtype), got)
    # accumulation in place; one fp32 addition more
    before = torch.randn(got.shape, generator=torch.Generator().manual_seed(2)).to(cuda_device)
    out = before.clone()
    assert moe.grouped_gemm_wgrad(g, x, s, e, out=out, accumulate=True) is out
    once = moe.grouped_gemm_wgrad(g, x, s, e)
    assert torch.equal(out, before + once)


@pytest.mark.gpu
@pytest.mark.parametrize('sizes,n,k', (
    ((4100,), 128, 128), ((4100,), 8, 264), ((20000,), 136, 8),
    ((63, 2000, 0, 513, 1), 300, 136), ((0, 0, 9000, 0), 128, 256),   # parts without rows, experts without rows
    ((0,), 128, 128), ((700, 1, 650) * 20, 128, 128), ((300,) * 37, 256, 256),
    ((800, 500), 1024, 1024),
), ids=str)
def test_wgrad_of_small_weights(cuda_device, sizes, n, k):
    """Few tiles: the rows of a group are split over a cluster of blocks, whose sums are added in the order of the parts."""
    from tilekernels_b200 import moe
    # (rows start on 16-byte boundaries)
    x, start, end, _ = _rows(sizes, -(-k // 8) * 8, cuda_device, gap=3, first=1)
    g, _, _, _ = _rows(sizes, -(-n // 8) * 8, cuda_device, gap=3, first=1, seed=1)
    x, g = x[:, :k], g[:, :n]
    s, e = int32(start, cuda_device), int32(end, cuda_device)
    for dtype in (torch.float32, torch.bfloat16):
        got = moe.grouped_gemm_wgrad(g, x, s, e, out_dtype=dtype)
        for i, (a, b) in enumerate(zip(start, end)):
            if a == b:
                assert (got[i] == 0).all()
            else:
                assert_product(got[i], g[a:b].cpu().double().T, x[a:b].cpu().double().T)
        assert torch.equal(moe.grouped_gemm_wgrad(g, x, s, e, out_dtype=dtype), got)
    before = torch.randn(got.shape, generator=torch.Generator().manual_seed(2)).to(cuda_device)
    out = before.clone()
    moe.grouped_gemm_wgrad(g, x, s, e, out=out, accumulate=True)
    assert torch.equal(out, before + moe.grouped_gemm_wgrad(g, x, s, e))


@pytest.mark.gpu
@pytest.mark.parametrize('sizes,n,k', (((40, 0), 1032, 2056), ((300, 200), 2048, 1160), ((4100,), 128, 136)), ids=str)
def test_accumulation_keeps_subnormals(cuda_device, sizes, n, k):
    """An addition in fp32 as it is defined, in whole tiles and in products that a cluster shares: a subnormal is kept where nothing
    is added to it, and counts where something is."""
    from tilekernels_b200 import moe
    start, end, used = segments(sizes)
    s, e = int32(start, cuda_device), int32(end, cuda_device)
    g = torch.zeros((used, -(-n // 8) * 8), dtype=torch.bfloat16, device=cuda_device)[:, :n]
    x = torch.zeros((used, k), dtype=torch.bfloat16, device=cuda_device)
    x[0] = 2.0 ** -63
    tiny = torch.tensor([1e-40, -1e-40, 2.0 ** -149, 2.0 ** -126, 0.0, 3.0], device=cuda_device)
    before = tiny[torch.arange(len(sizes) * n * k, device=cuda_device) % 6].view(len(sizes), n, k)
    out = before.clone()
    moe.grouped_gemm_wgrad(g, x, s, e, out=out, accumulate=True)
    assert torch.equal(out.view(torch.int32), before.view(torch.int32))
    g[0] = 2.0 ** -63   # every result of the first group is 2^-126
    moe.grouped_gemm_wgrad(g, x, s, e, out=out, accumulate=True)
    want = before.cpu().double()
    want[0] += 2.0 ** -126   # (exact in fp32 but for 3.0, which stays)
    assert torch.equal(out.cpu(), want.float())


@pytest.mark.gpu
@pytest.mark.parametrize('rows', (250, 1025, 9000))
def test_wgrad_of_long_groups_keeps_its_precision(cuda_device, rows):
    """The tensor core's sum goes on in registers every 256 rows.  A step of 16 rows cuts off at most one unit (2^-23 of the
    sum of magnitudes) per term and once for the accumulator, so 256 rows are off by at most 272 units; every addition in
    registers rounds by at most half a unit."""
    from tilekernels_b200 import moe
    n, k = 136, 264
    gen = torch.Generator().manual_seed(rows)
    g = (torch.rand((rows, n), generator=gen) + 0.5).to(torch.bfloat16).to(cuda_device)   # one sign: nothing averages out
    x = (torch.rand((rows, k), generator=gen) + 0.5).to(torch.bfloat16).to(cuda_device)
    got = moe.grouped_gemm_wgrad(g, x, int32([0], cuda_device), int32([rows], cuda_device))[0]
    want = g.double().T @ x.double()
    bound = (272 * 2.0 ** -23 + -(-rows // 256) * 2.0 ** -24) * want
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize('rows,n,k', ((9000, 2048, 2048), (80000, 136, 264)), ids=('whole', 'split'))
def test_wgrad_sums_of_one_sign_do_not_drift(cuda_device, rows, n, k):
    """What the tensor core cuts off has one sign, so it shows in the mean over all results.  Step t of the 16 between two additions
    in registers cuts off at most one unit (2^-23) of t / 16 of their sum: 8.5 units in all, where a sum left to the tensor core
    over 560 steps or more would lose some 280 (half a unit per step on average; 265 of 2^-23 were measured).  Additions in registers round
    either way; what is left of them in the mean is granted as much again."""
    from tilekernels_b200 import moe
    gen = torch.Generator(cuda_device).manual_seed(rows)
    g = (torch.rand((rows, n), generator=gen, device=cuda_device) + 0.5).to(torch.bfloat16)
    x = (torch.rand((rows, k), generator=gen, device=cuda_device) + 0.5).to(torch.bfloat16)
    before = torch.zeros((1, n, k), device=cuda_device)
    bounds = int32([0], cuda_device), int32([rows], cuda_device)
    want = g.double().T @ x.double()
    for got in (moe.grouped_gemm_wgrad(g, x, *bounds)[0], moe.grouped_gemm_wgrad(g, x, *bounds, out=before, accumulate=True)[0]):
        assert abs(((got.double() - want) / want).mean().item()) <= 17 * 2.0 ** -23


@pytest.mark.gpu
@pytest.mark.parametrize('sizes', ((300000,), (5, 20000, 0, 180000)), ids=str)
def test_bf16_wgrad_of_very_long_groups(cuda_device, sizes):
    """A sum of one sign over many rows, rounded to bf16: half a step of bf16, and before it what the sum itself is off by.  The tensor
    core adds up 4096 rows at most, 256 steps of 16 rows that cut off at most one unit (2^-23) of the accumulator and one of each of
    their products (2^-23 of the sum over one step, 1/256 of the sum); every addition in registers rounds by at most half a unit.
    Left to the tensor core alone, 300000 rows came out 1.9e-3 of the result further off."""
    from tilekernels_b200 import moe
    n, k = 1152, 1152
    start, end, used = segments(sizes, first=3)
    gen = torch.Generator(cuda_device).manual_seed(used)
    g = (torch.rand((used, n), generator=gen, device=cuda_device) + 0.5).to(torch.bfloat16)
    x = (torch.rand((used, k), generator=gen, device=cuda_device) + 0.5).to(torch.bfloat16)
    got = moe.grouped_gemm_wgrad(g, x, int32(start, cuda_device), int32(end, cuda_device), out_dtype=torch.bfloat16)
    for i, (a, b) in enumerate(zip(start, end)):
        want = torch.zeros((n, k), dtype=torch.float64, device=cuda_device)
        for r in range(a, b, 1 << 15):
            want += g[r:min(b, r + (1 << 15))].double().T @ x[r:min(b, r + (1 << 15))].double()
        bound = (272 * 2.0 ** -23 + -(-sizes[i] // 4096) * 2.0 ** -24) * want
        # half the distance of two bf16 numbers at `want`, or of the next binade where the sum may have reached it
        half = torch.exp2(torch.floor(torch.log2((want + bound).clamp(min=2.0 ** -100))) - 8)
        assert ((got[i].double() - want).abs() <= half + bound).all()


@pytest.mark.gpu
def test_gradients_against_differences(cuda_device):
    """The product is linear in either operand, and with small integers every sum is exact, so differences of the forward
    product have to equal the gradients to the last bit."""
    from tilekernels_b200 import moe
    gen = torch.Generator().manual_seed(6)
    sizes, n, k = (5, 0, 18, 40), 64, 32

    def ints(*shape):
        return torch.randint(-1, 2, shape, generator=gen).to(torch.bfloat16).to(cuda_device)

    start, end, used = segments(sizes)
    s, e = int32(start, cuda_device), int32(end, cuda_device)
    x, dx, c = ints(used, k), ints(used, k), ints(used, n)
    w, dw = ints(len(sizes), n, k), ints(len(sizes), n, k)

    def f(x, w):
        return (moe.grouped_gemm(x, w, s, e).double() * c.double()).sum().item()

    grad_x = moe.grouped_gemm(c, w, s, e, transpose_w=True).double()
    grad_w = moe.grouped_gemm_wgrad(c, x, s, e).double()
    assert f(x + dx, w) - f(x - dx, w) == 2 * (grad_x * dx.double()).sum().item()
    assert f(x, w + dw) - f(x, w - dw) == 2 * (grad_w * dw.double()).sum().item()


@pytest.mark.gpu
def test_bounds_outside_the_rows_are_clamped(cuda_device):
    from tilekernels_b200 import moe
    x, _, _, _ = _rows((20,), 64, cuda_device, spare=0)
    w = torch.ones((3, 32, 64), dtype=torch.bfloat16, device=cuda_device)
    s, e = int32([-5, 8, 30], cuda_device), int32([8, 1000, 7], cuda_device)
    got = moe.grouped_gemm(x, w, s, e)
    _check_groups(got, x.cpu().double(), w.cpu().double(), [0, 8], [8, 20])
    dw = moe.grouped_gemm_wgrad(x, x, s, e)
    assert_product(dw[0], x[:8].cpu().double().T, x[:8].cpu().double().T)
    assert_product(dw[1], x[8:].cpu().double().T, x[8:].cpu().double().T)
    assert (dw[2] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize('start,end,mine', (
    ((0, 5, 5), (10, 20, 12), ((0, 10), (10, 20), (20, 20))),           # overlapping
    ((12, 0, 14), (14, 8, 30), ((12, 14), (14, 14), (14, 30))),         # out of order
    ((40, -7, 3), (50, -9, 2), ((30, 30), (30, 30), (30, 30))),         # outside, ends before starts
    ((25, 0, 30, 10), (4, 10, 30, 20), ((0, 0), (0, 10), (10, 10), (10, 20))),  # experts without rows point elsewhere
    ((0,) * 40, (30,) * 40, ((0, 30),) + ((30, 30),) * 39),             # all the same
), ids=('overlapping', 'out of order', 'outside', 'empty', 'the same'))
def test_segments_that_overlap_or_go_back(cuda_device, start, end, mine):
    from tilekernels_b200 import moe
    x, _, _, _ = _rows((30,), 64, cuda_device, spare=0)
    w = torch.randn((len(start), 48, 64), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(cuda_device)
    s, e = int32(start, cuda_device), int32(end, cuda_device)
    first, last = zip(*mine)
    got = moe.grouped_gemm(x, w, s, e)
    _check_groups(got, x.cpu().double(), w.cpu().double(), first, last)
    member = torch.zeros(30, dtype=torch.bool)
    for a, b in mine:
        member[a:b] = True
    assert (got[~member.to(cuda_device)] == 0).all()
    dw = moe.grouped_gemm_wgrad(x, x, s, e)
    for i, (a, b) in enumerate(mine):
        if a == b:
            assert (dw[i] == 0).all()
        else:
            assert_product(dw[i], x[a:b].cpu().double().T, x[a:b].cpu().double().T)


@pytest.mark.gpu
def test_strided_operands(cuda_device):
    from tilekernels_b200 import moe
    sizes, n, k = (33, 0, 90), 136, 72
    start, end, used = segments(sizes)
    gen = torch.Generator().manual_seed(8)
    xs = torch.randn((used, k + 24), generator=gen).to(torch.bfloat16).to(cuda_device)
    ws = torch.randn((3, n + 5, k + 16), generator=gen).to(torch.bfloat16).to(cuda_device)
    x, w = xs[:, 8:8 + k], ws[:, 2:2 + n, 8:8 + k]
    s, e = int32(start, cuda_device), int32(end, cuda_device)
    _check_groups(moe.grouped_gemm(x, w, s, e), x.cpu().double(), w.cpu().double(), start, end)
    got = moe.grouped_gemm_wgrad(xs[:, 16:16 + 40], x, s, e)
    assert_product(got[2], xs[start[2]:end[2], 16:56].cpu().double().T, x[start[2]:end[2]].cpu().double().T)


@pytest.mark.gpu
def test_many_experts(cuda_device):
    from tilekernels_b200 import moe
    gen = torch.Generator().manual_seed(11)
    sizes = torch.randint(0, 4, (1024,), generator=gen).tolist()
    x, start, end, _ = _rows(sizes, 64, cuda_device)
    w = torch.randn((1024, 16, 64), generator=gen).to(torch.bfloat16).to(cuda_device)
    s, e = int32(start, cuda_device), int32(end, cuda_device)
    got = moe.grouped_gemm(x, w, s, e)
    _check_groups(got, x.cpu().double(), w.cpu().double(), start, end)
    dw = moe.grouped_gemm_wgrad(x, x, s, e)
    for i in range(0, 1024, 97):
        if sizes[i]:
            rows = x[start[i]:end[i]].cpu().double()
            assert_product(dw[i], rows.T, rows.T)


@pytest.mark.gpu
@pytest.mark.parametrize('form', (('e4m3', (1, 128), (128, 128)), ('e2m1', (1, 32), (1, 32)), ('nvfp4', (1, 16), (1, 16))), ids=lambda f: f[0])
def test_many_experts_with_many_rows(cuda_device, form):
    """More groups than a tile variant with large shared-memory needs has a table for."""
    from tilekernels_b200 import moe
    fmt, xb, wb = form
    experts, n, k = 130, 128, 128
    sizes = [(37 * i) % 140 for i in range(experts)]
    x, start, end, member = _rows(sizes, k, cuda_device)
    x[~member.to(cuda_device)] = 0
    xq, xv, xt = quantize(x, fmt, xb)
    w = torch.randn((experts * n, k), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda_device)
    wq, wv, wt = quantize(w, fmt, wb)
    alpha = xt * wt if fmt == 'nvfp4' else None
    got = moe.grouped_gemm(xq, (wq[0].view(experts, n, -1), wq[1]), int32(start, cuda_device), int32(end, cuda_device), xb, wb, alpha=alpha)
    _check_groups(got, xv, wv.view(experts, n, k), start, end, scale=None if alpha is None else [alpha.double().item()] * experts)


@pytest.mark.gpu
def test_no_rows(cuda_device):
    from tilekernels_b200 import moe
    w = torch.ones((2, 16, 64), dtype=torch.bfloat16, device=cuda_device)
    zero = int32([0, 0], cuda_device)
    empty = torch.empty((0, 64), dtype=torch.bfloat16, device=cuda_device)
    assert moe.grouped_gemm(empty, w, zero, zero).shape == (0, 16)
    assert (moe.grouped_gemm_wgrad(empty[:, :16], empty, zero, zero) == 0).all()
    out = torch.full((2, 16, 64), 2.0, device=cuda_device)
    moe.grouped_gemm_wgrad(empty[:, :16], empty, zero, zero, out=out, accumulate=True)
    assert (out == 2.0).all()
    # rows, but all of them of no expert
    x = torch.full((9, 64), float('nan'), dtype=torch.bfloat16, device=cuda_device)
    assert (moe.grouped_gemm(x, w, zero, zero) == 0).all()
    assert (moe.grouped_gemm_wgrad(x[:, :16], x, zero, zero) == 0).all()


@pytest.mark.gpu
def test_graph_follows_the_group_bounds(cuda_device):
    """Captured once, replayed with other rows and other segments: nothing about the groups is fixed at capture."""
    from tilekernels_b200 import moe
    n, k, rows = 200, 136, 400
    gen = torch.Generator().manual_seed(13)
    w = torch.randn((4, n, k), generator=gen).to(torch.bfloat16).to(cuda_device)
    x = torch.zeros((rows, k), dtype=torch.bfloat16, device=cuda_device)
    s, e = int32([0] * 4, cuda_device), int32([0] * 4, cuda_device)
    main = torch.zeros((4, n, k), device=cuda_device)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y = moe.grouped_gemm(x, w, s, e)
            dx = moe.grouped_gemm(y, w, s, e, transpose_w=True)
            moe.grouped_gemm_wgrad(y, x, s, e, out=main, accumulate=True)
    for sizes in ((100, 100, 100, 100), (0, 399, 0, 1), (7, 0, 0, 0)):
        start, end, _ = segments(sizes)
        new = torch.randn((rows, k), generator=gen).to(torch.bfloat16).to(cuda_device)
        with torch.cuda.stream(stream):
            x.copy_(new)
            s.copy_(int32(start, cuda_device))
            e.copy_(int32(end, cuda_device))
            main.zero_()
            graph.replay()
        torch.cuda.synchronize()
        _check_groups(y, x.cpu().double(), w.cpu().double(), start, end)
        _check_groups(dx, y.cpu().double(), w.cpu().double(), start, end, transpose=True)
        for i, (a, b) in enumerate(zip(start, end)):
            if a < b:
                assert_product(main[i], y[a:b].cpu().double().T, x[a:b].cpu().double().T)
        assert (y[sum(sizes):] == 0).all()


@pytest.mark.gpu
def test_expert_layer(cuda_device):
    """The way of a batch through quantized experts and back: expansion, up-projection, activation and cast, down-projection;
    then both products' gradients in bf16.  Every step is compared with 64 bits on the inputs it was given."""
    from tilekernels_b200 import moe, quant
    from test_block_scaled_gemm import PACKED
    gen = torch.Generator().manual_seed(21)
    tokens, hidden, inter, experts, topk, align = 60, 512, 256, 4, 2, 16
    x = torch.randn((tokens, hidden), generator=gen).to(torch.bfloat16).to(cuda_device)
    choice = torch.stack([torch.randperm(experts, generator=gen)[:topk] for _ in range(tokens)])
    order, start, end, at = [], [], [], 0
    for e in range(experts):
        mine = (choice == e).nonzero().tolist()
        start.append(at)
        end.append(at + len(mine))
        order.append(mine)
        at = -(-end[-1] // align) * align
    t2p = torch.full((tokens, topk), -1, dtype=torch.int32)
    p2e = torch.full((at,), -1, dtype=torch.int32)
    for e in range(experts):
        for i, (t, j) in enumerate(order[e]):
            t2p[t, j] = start[e] + i
            p2e[start[e] + i] = e
    t2p, p2e = t2p.to(cuda_device), p2e.to(cuda_device)
    s, e = int32(start, cuda_device), int32(end, cuda_device)
    w1 = (torch.randn((experts, 2 * inter, hidden), generator=gen) * 0.05).to(torch.bfloat16).to(cuda_device)
    w2 = (torch.randn((experts, hidden, inter), generator=gen) * 0.05).to(torch.bfloat16).to(cuda_device)
    w1q = quant.per_block_cast(w1.view(-1, hidden), 'e4m3', (128, 128), **PACKED)
    w2q = quant.per_block_cast(w2.view(-1, inter), 'e4m3', (128, 128), **PACKED)
    w1v = dequantized(*w1q, (128, 128)).view(w1.shape)
    w2v = dequantized(*w2q, (128, 128)).view(w2.shape)

    q, sf = quant.per_token_cast(x, 'e4m3', 128, None, True, True, True)
    xq = moe.expand_to_fused_with_sf((q, sf.contiguous()), 128, t2p, p2e, True)
    up = moe.grouped_gemm(xq, (w1q[0].view(w1.shape), w1q[1]), s, e, (1, 128), (128, 128))
    _check_groups(up, dequantized(*xq, (1, 128)), w1v, start, end)
    act = quant.swiglu_forward_and_per_token_cast(up, 'e4m3', 128, pos_to_expert=p2e, **PACKED)
    down = moe.grouped_gemm(act, (w2q[0].view(w2.shape), w2q[1]), s, e, (1, 128), (128, 128))
    _check_groups(down, dequantized(*act, (1, 128)), w2v, start, end)
    assert (down[p2e < 0] == 0).all()

    xe = moe.expand_to_fused(x, t2p, p2e)
    d_up = torch.randn(up.shape, generator=gen).to(torch.bfloat16).to(cuda_device)
    dx = moe.grouped_gemm(d_up, w1, s, e, transpose_w=True)
    dw1 = moe.grouped_gemm_wgrad(d_up, xe, s, e)
    _check_groups(dx, d_up.cpu().double(), w1.cpu().double(), start, end, transpose=True)
    for i in range(experts):
        rows = slice(start[i], end[i])
        assert_product(dw1[i], d_up[rows].cpu().double().T, xe[rows].cpu().double().T)


@pytest.mark.gpu
def test_refusals(cuda_device):
    from tilekernels_b200 import moe
    x = torch.zeros((8, 64), dtype=torch.bfloat16, device=cuda_device)
    w = torch.zeros((2, 32, 64), dtype=torch.bfloat16, device=cuda_device)
    s, e = int32([0, 4], cuda_device), int32([4, 8], cuda_device)
    for args, kw in (
        ((x.float(), w, s, e), {}), ((x, w.half(), s, e), {}), ((x[:, :32], w, s, e), {}), ((x, w, s[:1], e), {}), ((x, w, s.long(), e), {}),
        ((x, w, s.cpu(), e), {}), ((x, w[0], s, e), {}), ((x, w, s, e), dict(alpha=torch.ones(1, device=cuda_device))),
        ((x, w, s, e), dict(x_block_size=(1, 128))), ((x.T, w, s, e), {}), ((x, w, s, e), dict(transpose_w=True)),
        ((x, w, s, e), dict(out=torch.empty((8, 33), dtype=torch.bfloat16, device=cuda_device))),
        (((x.view(torch.int8), s), (w.view(torch.int8), s), s, e), dict(x_block_size=(1, 32), w_block_size=(1, 32), transpose_w=True)),
    ):
        with pytest.raises(AssertionError):
            moe.grouped_gemm(*args, **kw)
    with pytest.raises(RuntimeError, match='16-byte'):
        moe.grouped_gemm(torch.zeros((8, 68), dtype=torch.bfloat16, device=cuda_device)[:, :64], w, s, e)
    with pytest.raises(RuntimeError, match='1024'):
        many = torch.zeros(1025, dtype=torch.int32, device=cuda_device)
        moe.grouped_gemm_wgrad(x, x, many, many)
    for args, kw in (
        ((x.float(), x, s, e), {}), ((x[:4], x, s, e), {}), ((x, x, s, e), dict(out_dtype=torch.float16)), ((x, x, s, e), dict(accumulate=True)),
        ((x, x, s, e), dict(out=torch.empty((2, 64, 64), dtype=torch.bfloat16, device=cuda_device))),
        ((x, x, s, e), dict(out_dtype=torch.bfloat16, accumulate=True, out=torch.empty((2, 64, 64), dtype=torch.bfloat16, device=cuda_device))),
    ):
        with pytest.raises(AssertionError):
            moe.grouped_gemm_wgrad(*args, **kw)


def test_cpu_tensors_are_refused():
    from tilekernels_b200 import moe
    x, w = torch.zeros((8, 64), dtype=torch.bfloat16), torch.zeros((2, 32, 64), dtype=torch.bfloat16)
    bounds = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(AssertionError):
        moe.grouped_gemm(x, w, bounds, bounds)
    with pytest.raises(AssertionError):
        moe.grouped_gemm_wgrad(x, x, bounds, bounds)
