"""block_scaled_gemm against the product of the dequantised operands in 64 bits."""
import pytest
import torch

from product_helpers import assert_product, dequantized

PACKED = dict(use_tma_aligned_col_major_sf=True, round_sf=True, use_packed_ue8m0=True)
# (name, blocks of a, blocks of b)
FORMS = (('e4m3', (1, 128), (128, 128)), ('e4m3', (1, 128), (1, 128)), ('e4m3', (1, 32), (1, 32)), ('e4m3', (1, 32), (128, 128)),
         ('e4m3', (1, 128), (32, 32)), ('e2m1', (1, 32), (1, 32)), ('e2m1', (1, 32), (32, 32)), ('nvfp4', (1, 16), (1, 16)))


def _id(form):
    return f'{form[0]}-{form[1][0]}x{form[1][1]}-{form[2][0]}x{form[2][1]}'


def quantize(x, fmt, block):
    """(operand, 64-bit values) of x, quantized by the casts."""
    from tilekernels_b200 import quant
    if fmt == 'nvfp4':
        ts = (x.float().abs().max() / 2688).reshape(1)
        op = quant.per_token_cast_to_nvfp4(x, ts)
        return op, dequantized(*op, block), ts
    if block[0] == 1:
        op = quant.per_token_cast(x, fmt, block[1], None, *PACKED.values())
    else:
        op = quant.per_block_cast(x, fmt, block, **PACKED)
    return op, dequantized(*op, block), None


def _matrices(m, n, k, device, seed=0):
    gen = torch.Generator().manual_seed(seed + m * 7 + n * 3 + k)
    a = torch.randn((m, k), generator=gen)
    a *= torch.exp2(torch.randint(-6, 7, (m, (k + 31) // 32), generator=gen).float()).repeat_interleave(32, 1)[:, :k]   # scales differ
    b = torch.randn((n, k), generator=gen) * torch.exp2(torch.randint(-6, 7, (n, 1), generator=gen).float())
    return a.to(torch.bfloat16).to(device), b.to(torch.bfloat16).to(device)


@pytest.mark.gpu
@pytest.mark.parametrize('form', FORMS, ids=_id)
@pytest.mark.parametrize('m,n,k', ((1, 128, 128), (1, 8, 64), (5, 4096, 1024), (31, 136, 576), (33, 257, 320), (128, 64, 2048),
                                   (129, 1000, 704), (500, 520, 1088), (1027, 384, 512)))
def test_against_64_bits(cuda_device, form, m, n, k):
    from tilekernels_b200 import quant
    fmt, ab, bb = form
    a, b = _matrices(m, n, k, cuda_device)
    (qa, va, ta), (qb, vb, tb) = quantize(a, fmt, ab), quantize(b, fmt, bb)
    alpha = ta * tb if fmt == 'nvfp4' else None
    got = quant.block_scaled_gemm(qa, qb, ab, bb, alpha=alpha)
    assert got.shape == (m, n) and got.dtype == torch.bfloat16 and got.is_contiguous()
    assert_product(got, va, vb, 1.0 if alpha is None else alpha.double().item())
    # the same call again gives the same bits
    assert torch.equal(quant.block_scaled_gemm(qa, qb, ab, bb, alpha=alpha), got)


@pytest.mark.gpu
@pytest.mark.parametrize('form', FORMS, ids=_id)
@pytest.mark.parametrize('m,n,k', ((1, 200, 7168), (16, 8, 16384), (31, 129, 4096), (33, 264, 6400), (64, 1024, 3328), (65, 100, 12288)))
def test_few_tiles_and_a_long_k(cuda_device, form, m, n, k):
    """Products that several blocks share along k, down to the last columns of the last part."""
    from tilekernels_b200 import quant
    fmt, ab, bb = form
    a, b = _matrices(m, n, k, cuda_device)
    (qa, va, ta), (qb, vb, tb) = quantize(a, fmt, ab), quantize(b, fmt, bb)
    alpha = ta * tb if fmt == 'nvfp4' else None
    got = quant.block_scaled_gemm(qa, qb, ab, bb, alpha=alpha)
    assert_product(got, va, vb, 1.0 if alpha is None else alpha.double().item())
    for _ in range(3):
        assert torch.equal(quant.block_scaled_gemm(qa, qb, ab, bb, alpha=alpha), got)


@pytest.mark.gpu
@pytest.mark.parametrize('form', FORMS, ids=_id)
def test_many_waves(cuda_device, form):
    """Several tiles per block, whose scales differ from block to block along k: every sum against 64 bits, on the device."""
    from tilekernels_b200 import quant
    fmt, ab, bb = form
    m, n, k = 3000, 2600, 2048
    a, b = _matrices(m, n, k, cuda_device)
    (qa, va, ta), (qb, vb, tb) = quantize(a, fmt, ab), quantize(b, fmt, bb)
    alpha = ta * tb if fmt == 'nvfp4' else torch.ones(1, device=cuda_device)
    va, vb = va.to(cuda_device) * alpha.double(), vb.to(cuda_device)
    want, magnitudes = va @ vb.T, va.abs() @ vb.abs().T
    bound = k * 2.0 ** -23 * magnitudes
    bound += 2.0 ** -8 * (want.abs() + bound)
    for _ in range(3):
        got = quant.block_scaled_gemm(qa, qb, ab, bb, alpha=alpha)
        assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize('m', (1, 300))
def test_alpha_out_and_strides(cuda_device, m):
    from tilekernels_b200 import quant
    n, k = 264, 512
    a, b = _matrices(m, n, k, cuda_device)
    for fmt, block in (('e4m3', (1, 32)), ('e2m1', (1, 32))):
        (qa, va, _), (qb, vb, _) = quantize(a, fmt, block), quantize(b, fmt, block)
        alpha = torch.full((1,), -0.75, device=cuda_device)
        for width, first in ((n, 0), (n + 8, 8), (n + 7, 3), (n + 6, 2)):   # rows on any boundary, columns beside left alone
            store = torch.full((m + 2, width), 7.0, dtype=torch.bfloat16, device=cuda_device)
            out = store[1:-1, first:first + n]
            assert quant.block_scaled_gemm(qa, qb, block, block, alpha=alpha, out=out) is out
            assert_product(out, va, vb, -0.75)
            keep = torch.ones_like(store, dtype=torch.bool)
            keep[1:-1, first:first + n] = False
            assert (store[keep] == 7.0).all()
        # data in the middle of wider rows, scales of another pitch
        data = torch.zeros((m, qa[0].shape[1] + 48), dtype=torch.uint8, device=cuda_device).view(qa[0].dtype)
        data[:, 16:16 + qa[0].shape[1]] = qa[0]
        sf = torch.zeros((qa[1].shape[0], qa[1].shape[1] + 3), dtype=torch.int32, device=cuda_device)[:, :qa[1].shape[1]].copy_(qa[1])
        got = quant.block_scaled_gemm((data[:, 16:16 + qa[0].shape[1]], sf), qb, block, block)
        assert_product(got, va, vb)


@pytest.mark.gpu
@pytest.mark.parametrize('fmt,block', (('e4m3', (128, 128)), ('e4m3', (32, 32)), ('e4m3', (32, 128)), ('e2m1', (32, 32)), ('e2m1', (128, 32))))
@pytest.mark.parametrize('m', (7, 130, 400))
def test_scales_of_row_blocks_in_the_left_operand(cuda_device, fmt, block, m):
    from tilekernels_b200 import quant
    a, b = _matrices(m, 200, 576, cuda_device)
    other = (1, 128) if fmt == 'e4m3' else (1, 32)
    (qa, va, _), (qb, vb, _) = quantize(a, fmt, block), quantize(b, fmt, other)
    assert_product(quant.block_scaled_gemm(qa, qb, block, other), va, vb)


@pytest.mark.gpu
def test_extreme_scales_and_special_codes(cuda_device):
    """Scales of 2^-60 .. 2^60 in either operand, and rows whose NaN reaches their own results only."""
    from tilekernels_b200 import quant
    m, n, k = 70, 200, 256
    gen = torch.Generator().manual_seed(4)
    a, b = torch.randn((m, k), generator=gen), torch.randn((n, k), generator=gen)
    a *= torch.exp2(torch.linspace(-60, 60, m).round())[:, None]
    b *= torch.exp2(torch.linspace(60, -60, n).round())[:, None] * 2.0 ** -10
    (qa, va, _), (qb, vb, _) = quantize(a.to(cuda_device), 'e4m3', (1, 32)), quantize(b.to(cuda_device), 'e4m3', (1, 32))
    assert_product(quant.block_scaled_gemm(qa, qb, (1, 32), (1, 32)), va, vb)
    bytes_ = qa[0].clone().view(torch.uint8)
    bytes_[3, 5] = 0x7f   # NaN
    got = quant.block_scaled_gemm((bytes_.view(torch.float8_e4m3fn), qa[1]), qb, (1, 32), (1, 32))
    assert torch.isnan(got[3]).all() and torch.isfinite(got[:3]).all() and torch.isfinite(got[4:]).all()


@pytest.mark.gpu
def test_empty(cuda_device):
    from tilekernels_b200 import quant
    a, b = _matrices(4, 64, 128, cuda_device)
    qa, qb = quantize(a, 'e4m3', (1, 128))[0], quantize(b, 'e4m3', (1, 128))[0]
    empty = (qa[0][:0], qa[1][:0])
    assert quant.block_scaled_gemm(empty, qb, (1, 128), (1, 128)).shape == (0, 64)
    assert quant.block_scaled_gemm(qa, empty, (1, 128), (1, 128)).shape == (4, 0)


@pytest.mark.gpu
def test_streams_and_graphs(cuda_device):
    """Work goes to the caller's stream, and a captured call reads what its buffers hold when it is replayed; two graphs
    replayed on two streams do not disturb each other."""
    from tilekernels_b200 import quant
    m, n, k = 300, 512, 1024
    inputs = [_matrices(m, n, k, cuda_device, seed) for seed in range(4)]
    want = []
    for a, b in inputs:
        qa, qb = quantize(a, 'e2m1', (1, 32))[0], quantize(b, 'e2m1', (1, 32))[0]
        want.append((qa, qb, quant.block_scaled_gemm(qa, qb, (1, 32), (1, 32)).clone()))
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        (da, sa), (db, sb), _ = want[i]
        # (clones keep the column-major strides of the scales)
        buffers = [da.clone(), sa.clone(), db.clone(), sb.clone()]
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = quant.block_scaled_gemm((buffers[0], buffers[1]), (buffers[2], buffers[3]), (1, 32), (1, 32))
        graphs.append((graph, stream, buffers, out))
    for turn in (2, 0):
        for i, (graph, stream, buffers, out) in enumerate(graphs):
            with torch.cuda.stream(stream):
                (da, sa), (db, sb), _ = want[turn + i]
                for dst, src in zip(buffers, (da, sa, db, sb)):
                    dst.copy_(src)
                graph.replay()
        torch.cuda.synchronize()
        for i, (_, _, _, out) in enumerate(graphs):
            assert torch.equal(out, want[turn + i][2])


@pytest.mark.gpu
def test_refusals(cuda_device):
    from tilekernels_b200 import quant
    a, b = _matrices(8, 64, 256, cuda_device)
    qa, qb = quantize(a, 'e4m3', (1, 128))[0], quantize(b, 'e4m3', (1, 128))[0]
    fa = quantize(a, 'e2m1', (1, 32))[0]
    nv = quantize(a, 'nvfp4', (1, 16))[0]
    f32 = quant.per_token_cast(a, 'e4m3', 128, None, True, True, False)
    bad = (
        (fa, qb, (1, 32), (1, 128), {}),                                   # two formats
        (f32, qb, (1, 128), (1, 128), {}),                                 # fp32 scales
        (qa, qb, (1, 32), (1, 128), {}),                                   # scales of another block size
        (qa, qb, (1, 64), (1, 128), {}),
        (qa, (qb[0][:, :128], qb[1]), (1, 128), (1, 128), {}),             # inner sizes
        (qa, (qb[0], qb[1][:60]), (1, 128), (1, 128), {}),                 # too few scales
        (nv, fa, (1, 16), (1, 32), {}),                                    # e4m3 with ue8m0 scales
        (qa, qb, (1, 128), (1, 128), dict(alpha=torch.ones(2, device=cuda_device))),
        (qa, qb, (1, 128), (1, 128), dict(alpha=torch.ones(1))),
        (qa, qb, (1, 128), (1, 128), dict(out=torch.empty((8, 64), device=cuda_device))),
        (qa, qb, (1, 128), (1, 128), dict(out=torch.empty((8, 65), dtype=torch.bfloat16, device=cuda_device))),
        ((qa[0].cpu(), qa[1].cpu()), qb, (1, 128), (1, 128), {}),
    )
    for x, w, xb, wb, kw in bad:
        with pytest.raises(AssertionError):
            quant.block_scaled_gemm(x, w, xb, wb, **kw)
    with pytest.raises(RuntimeError, match='multiple of 32'):
        quant.block_scaled_gemm((qa[0][:, :144], qa[1]), (qb[0][:, :144], qb[1]), (1, 128), (1, 128))
    wide = torch.zeros((8, 264), dtype=torch.uint8, device=cuda_device).view(torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match='16-byte'):
        quant.block_scaled_gemm((wide[:, :256], qa[1]), qb, (1, 128), (1, 128))


def test_cpu_tensors_are_refused():
    from tilekernels_b200 import quant
    x = (torch.zeros((4, 128), dtype=torch.int8), torch.zeros((4, 2), dtype=torch.int32))
    with pytest.raises(AssertionError):
        quant.block_scaled_gemm(x, x, (1, 32), (1, 32))
