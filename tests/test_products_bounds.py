"""Where the products and the NVFP4 cast write: outputs inside larger buffers whose every other byte has to stay, and tensors
whose element offsets pass 32 bits."""
import pytest
import torch

from product_helpers import assert_product, dequantized, int32
from test_block_scaled_gemm import quantize

pytestmark = pytest.mark.gpu


def _guarded(shape, dtype, device, pad=4096):
    """A contiguous tensor in the middle of a byte buffer filled with 0xA5, and a check of the bytes around it."""
    size = torch.empty((), dtype=dtype).element_size()
    n = size
    for d in shape:
        n *= d
    store = torch.full((n + 2 * pad,), 0xA5, dtype=torch.uint8, device=device)
    inner = store[pad:pad + n].view(dtype).view(shape)

    def check():
        assert (store[:pad] == 0xA5).all() and (store[pad + n:] == 0xA5).all()
    return inner, check


@pytest.mark.parametrize('rows', (1, 31, 33, 129, 300))
@pytest.mark.parametrize('n', (8, 129, 200, 257))
def test_products_write_their_output_only(cuda_device, rows, n):
    from tilekernels_b200 import moe, quant
    gen = torch.Generator().manual_seed(rows * n)
    x = torch.randn((rows, 128), generator=gen).to(torch.bfloat16).to(cuda_device)
    w = torch.randn((n, 128), generator=gen).to(torch.bfloat16).to(cuda_device)
    for fmt, block in (('e4m3', (1, 128)), ('e2m1', (1, 32)), ('nvfp4', (1, 16))):
        (qx, xv, _), (qw, wv, _) = quantize(x, fmt, block), quantize(w, fmt, block)
        out, check = _guarded((rows, n), torch.bfloat16, cuda_device)
        quant.block_scaled_gemm(qx, qw, block, block, out=out)
        check()
        assert_product(out, xv, wv)
    s, e = int32([0, rows // 2], cuda_device), int32([rows // 2, rows], cuda_device)
    out, check = _guarded((rows, n), torch.bfloat16, cuda_device)
    moe.grouped_gemm(x, w.expand(2, n, 128).contiguous(), s, e, out=out)
    check()
    assert_product(out, x.cpu().double(), w.cpu().double())
    if n % 8 == 0:
        g = torch.randn((rows, n), generator=gen).to(torch.bfloat16).to(cuda_device)
        for dtype, accumulate in ((torch.float32, False), (torch.bfloat16, False), (torch.float32, True)):
            out, check = _guarded((2, n, 128), dtype, cuda_device)
            if accumulate:
                out.zero_()
            moe.grouped_gemm_wgrad(g, x, s, e, out_dtype=dtype, out=out, accumulate=accumulate)
            check()
            assert_product(out[1], g[rows // 2:].cpu().double().T, x[rows // 2:].cpu().double().T)


@pytest.mark.parametrize('n,k', ((8, 8), (129, 131), (1, 300), (257, 5)))
@pytest.mark.parametrize('dtype', (torch.float32, torch.bfloat16), ids=('fp32', 'bf16'))
def test_split_weight_gradients_write_their_output_only(cuda_device, n, k, dtype):
    """Long groups of a small weight, whose rows a cluster shares: eager, on two streams at once, and replayed with other bounds."""
    from tilekernels_b200 import moe
    gen = torch.Generator().manual_seed(n * k)
    rows = 5000
    g = torch.randn((rows, -(-n // 8) * 8), generator=gen).to(torch.bfloat16).to(cuda_device)[:, :n]
    x = torch.randn((rows, -(-k // 8) * 8), generator=gen).to(torch.bfloat16).to(cuda_device)[:, :k]
    s, e = int32([3, 1500], cuda_device), int32([1500, 4999], cuda_device)

    def check_values(out, bounds):
        for i, (a, b) in enumerate(bounds):
            assert_product(out[i], g[a:b].cpu().double().T, x[a:b].cpu().double().T)

    out, check = _guarded((2, n, k), dtype, cuda_device)
    moe.grouped_gemm_wgrad(g, x, s, e, out_dtype=dtype, out=out)
    check()
    check_values(out, ((3, 1500), (1500, 4999)))
    want = out.clone()
    streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
    outs = [_guarded((2, n, k), dtype, cuda_device) for _ in streams]
    torch.cuda.synchronize(cuda_device)
    for _ in range(5):
        for stream, (o, _) in zip(streams, outs):
            with torch.cuda.stream(stream):
                moe.grouped_gemm_wgrad(g, x, s, e, out_dtype=dtype, out=o)
    torch.cuda.synchronize(cuda_device)
    for o, c in outs:
        c()
        assert torch.equal(o, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moe.grouped_gemm_wgrad(g, x, s, e, out_dtype=dtype, out=out)
    s.copy_(int32([0, 4000], cuda_device))
    e.copy_(int32([17, 5000], cuda_device))
    graph.replay()
    check()
    check_values(out, ((0, 17), (4000, 5000)))


@pytest.mark.parametrize('mode', ('bf16', 'fp32', 'accumulate'))
@pytest.mark.parametrize('n,k', ((1290, 1165), (1, 9500), (2049, 600)))
def test_whole_weight_gradients_write_their_output_only(cuda_device, mode, n, k):
    """Weights whose tiles fill the SMs, so that no group is split, in a call of more than 16384 rows; rows of no group hold NaN."""
    from tilekernels_b200 import moe
    gen = torch.Generator(cuda_device).manual_seed(n * k)
    rows, bounds = 16500, ((2, 4200), (4200, 4200), (4207, 16497))
    g = torch.randn((rows, -(-n // 8) * 8), generator=gen, device=cuda_device).to(torch.bfloat16)[:, :n]
    x = torch.randn((rows, -(-k // 8) * 8), generator=gen, device=cuda_device).to(torch.bfloat16)[:, :k]
    for a, b in ((0, 2), (4200, 4207), (16497, rows)):
        g[a:b] = float('nan')
        x[a:b] = float('inf')
    s, e = (int32(list(v), cuda_device) for v in zip(*bounds))
    dtype = torch.bfloat16 if mode == 'bf16' else torch.float32
    out, check = _guarded((3, n, k), dtype, cuda_device)
    if mode == 'accumulate':
        out.zero_()
    moe.grouped_gemm_wgrad(g, x, s, e, out_dtype=dtype, out=out, accumulate=mode == 'accumulate')
    check()
    for i, (a, b) in enumerate(bounds):
        a64, b64 = g[a:b].double(), x[a:b].double()
        want, bound = a64.T @ b64, (b - a) * 2.0 ** -23 * (a64.abs().T @ b64.abs())
        if mode == 'bf16':
            bound += 2.0 ** -8 * (want.abs() + bound)
        assert ((out[i].double() - want).abs() <= bound).all()


@pytest.mark.parametrize('rows,hidden', ((1, 16), (3, 528), (129, 1040)))
@pytest.mark.parametrize('dtype', (torch.bfloat16, torch.float32), ids=('bf16', 'fp32'))
def test_nvfp4_writes_its_output_only(cuda_device, rows, hidden, dtype):
    from tilekernels_b200 import _lib, quant
    x = torch.randn((rows, hidden), generator=torch.Generator().manual_seed(hidden)).to(dtype).to(cuda_device)
    ts = torch.full((1,), 0.001, device=cuda_device)
    code = _lib.DT_BF16 if dtype is torch.bfloat16 else _lib.DT_FP32
    stream = torch.cuda.current_stream(cuda_device).cuda_stream
    q, check_q = _guarded((rows, hidden // 2), torch.int8, cuda_device)
    sf, check_sf = _guarded((rows, hidden // 16), torch.float8_e4m3fn, cuda_device)
    back, check_back = _guarded((rows, hidden), dtype, cuda_device)
    assert _lib.lib().tkq_per_token_cast_nvfp4(x.data_ptr(), code, rows, hidden, hidden, ts.data_ptr(), q.data_ptr(), sf.data_ptr(), stream) == 0
    assert _lib.lib().tkq_cast_back_nvfp4(q.data_ptr(), sf.data_ptr(), ts.data_ptr(), rows, hidden, code, back.data_ptr(), stream) == 0
    for check in (check_q, check_sf, check_back):
        check()
    want = quant.per_token_cast_to_nvfp4(x, ts)
    assert torch.equal(q, want[0]) and torch.equal(sf.view(torch.uint8), want[1].view(torch.uint8))
    assert torch.equal(back, quant.cast_back(want, 'bf16' if dtype is torch.bfloat16 else 'fp32', (1, 16), tensor_scale=ts))


def test_offsets_beyond_32_bits(cuda_device):
    """Outputs, weights and inputs of more than 2^31 elements; what lies behind that mark is compared."""
    from tilekernels_b200 import moe, quant
    gen = torch.Generator('cuda').manual_seed(2)

    def rand(*shape):
        return torch.randn(shape, generator=gen, device=cuda_device, dtype=torch.bfloat16)

    rows, n, k = 66001, 32768, 64   # 2.16e9 results
    x, w = rand(rows, k), rand(1, n, k)
    out = moe.grouped_gemm(x, w, int32([5], cuda_device), int32([rows], cuda_device))
    assert_product(out[-3:], x[-3:].cpu().double(), w[0].cpu().double())
    assert (out[:5] == 0).all()
    (qx, xv, _), (qw, wv, _) = quantize(x, 'e4m3', (1, 32)), quantize(w[0], 'e4m3', (1, 32))
    quant.block_scaled_gemm(qx, qw, (1, 32), (1, 32), out=out)
    assert_product(out[-3:], xv[-3:], wv)
    del out, qx, qw
    experts, n, k = 33, 8192, 8192   # 2.2e9 weights
    w = rand(experts, n, k)
    start = int32(list(range(experts)), cuda_device)
    end = start + 1
    x = rand(experts, k)
    for transpose in (False, True):
        got = moe.grouped_gemm(x, w, start, end, transpose_w=transpose)
        last = w[-1].T if transpose else w[-1]
        assert_product(got[-1:], x[-1:].cpu().double(), last.cpu().double())
    g = rand(experts, n)
    moe.grouped_gemm_wgrad(g, x, start, end, out_dtype=torch.bfloat16, out=w)
    assert_product(w[-1], g[-1:].cpu().double().T, x[-1:].cpu().double().T)
    del w
    x = rand(300001, 7168)   # 2.15e9 values
    ts = torch.full((1,), 0.002, device=cuda_device)
    q, sf = quant.per_token_cast_to_nvfp4(x, ts)
    want = quant.per_token_cast_to_nvfp4(x[-2:].contiguous(), ts)
    assert torch.equal(q[-2:], want[0]) and torch.equal(sf[-2:].view(torch.uint8), want[1].view(torch.uint8))
    del x
    back = quant.cast_back((q, sf), 'bf16', (1, 16), tensor_scale=ts)
    assert torch.equal(back[-2:], quant.cast_back(want, 'bf16', (1, 16), tensor_scale=ts))
    assert torch.equal(back[-2:].cpu().double(), (dequantized(*want, (1, 16)) * ts.double().item()).float().bfloat16().double())
