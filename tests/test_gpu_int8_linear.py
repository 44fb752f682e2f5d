"""GPU tests of the 8-bit linear layer against its definition in 64 bits: codes exactly, products within the rounding of
the fp32 scaling and of the output."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(autouse=True)
def no_device_error():
    from tilemix_b200.attention.tilemix import device_error_code

    if torch.cuda.is_available():
        device_error_code()
    yield
    if torch.cuda.is_available():
        assert device_error_code() == 0


def _codes_of(x):
    """Codes and scales by their definition in 64 bits (127 x / amax is exact enough there to tell every tie)."""
    d = x.double().cpu().numpy()
    amax = np.abs(d).max(1, keepdims=True)
    q = np.divide(127 * d, amax, out=np.zeros_like(d), where=amax > 0)
    return np.trunc(q + 0.5 * np.sign(q)), amax[:, 0] / 127


def _operands(dev, m, n, k, seed):
    """Random codes in rows padded to 16 bytes, the padding filled with what must not be read."""
    g = torch.Generator().manual_seed(seed)
    wide = (k + 15) // 16 * 16
    x8 = torch.randint(-127, 128, (m, wide), generator=g, dtype=torch.int8).to(dev)[:, :k]
    w8 = torch.randint(-127, 128, (n, wide), generator=g, dtype=torch.int8).to(dev)[:, :k]
    xs, ws = torch.rand(m, generator=g).to(dev) * 1e-3, torch.rand(n, generator=g).to(dev) * 1e-2
    return x8, xs, w8, ws


def _check(out, x8, xs, w8, ws, bias=None):
    """fp32: the int32 sum is rounded once, each scale and the bias' sum once more; then the output's own rounding."""
    exact = x8.double() @ w8.double().t()
    scaled = exact * xs.double()[:, None] * ws.double()
    ref = scaled if bias is None else scaled + bias.double()
    # below fp16's normal range the output's step is 2^-24
    bound = scaled.abs() * 3 * 2.0 ** -24 + ref.abs() * (2.0 ** -24 + HALF_STEP[out.dtype]) * 1.001 + 2.0 ** -25
    err = (out.double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


SHAPES = [(1, 64, 64), (1, 1, 1), (2, 130, 100), (16, 4096, 512), (17, 257, 129), (33, 500, 2048), (64, 1024, 4096),
          (65, 136, 3000), (128, 384, 640), (129, 100, 1000), (200, 1, 33), (300, 777, 1111), (513, 2050, 256),
          (1000, 4096, 300), (2100, 5000, 520), (1, 8192, 16384), (48, 33, 20000)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_matmul_matches_exact_sums(cuda_device, m, n, k, dtype):
    from tilemix_b200.linear.int8_linear import int8_matmul

    x8, xs, w8, ws = _operands(cuda_device, m, n, k, seed=m + n + k)
    _check(int8_matmul(x8, xs, w8, ws, out_dtype=dtype), x8, xs, w8, ws)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(1)).to(cuda_device, dtype)
    _check(int8_matmul(x8, xs, w8, ws, bias, out_dtype=dtype), x8, xs, w8, ws, bias)


def test_largest_sums_do_not_wrap(cuda_device):
    from tilemix_b200.linear.int8_linear import int8_matmul

    k = 131071
    wide = (k + 15) // 16 * 16
    x8 = torch.full((3, wide), 127, dtype=torch.int8, device=cuda_device)[:, :k]
    w8 = torch.full((5, wide), -128, dtype=torch.int8, device=cuda_device)[:, :k]
    xs, ws = torch.full((3,), 1e-4, device=cuda_device), torch.ones(5, device=cuda_device)
    _check(int8_matmul(x8, xs, w8, ws, out_dtype=torch.float32), x8, xs, w8, ws)


def test_a_token_does_not_depend_on_its_batch(cuda_device):
    """Every launch shape gives the same bits."""
    from tilemix_b200.linear.int8_linear import int8_matmul

    x8, xs, w8, ws = _operands(cuda_device, 1500, 1000, 4000, seed=3)
    bias = torch.randn(1000, generator=torch.Generator().manual_seed(2)).to(cuda_device, torch.float16)
    full = int8_matmul(x8, xs, w8, ws, bias)
    for m in (1, 16, 31, 64, 100, 129, 400, 1499):
        assert torch.equal(int8_matmul(x8[:m], xs[:m], w8, ws, bias), full[:m]), m


def _rows(m, k, seed, dtype):
    x = torch.randn((m, k), generator=torch.Generator().manual_seed(seed))
    x *= torch.exp2(torch.arange(m) % 9 - 4.0)[:, None]
    if k > 4:
        x[:, 3] *= 40
        x[0, 1], x[0, 2] = x[0].abs().max(), x[0].abs().max() / 2  # 127 and the tie 63.5
    if m > 2:
        x[2] = 0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k", [(1, 1), (5, 8), (3, 100), (4, 2048), (7, 4096), (3, 5000), (2, 16384), (3, 16392),
                                 (2, 40001)])
def test_quantiser_matches_its_definition(cuda_device, m, k, dtype):
    from tilemix_b200.linear.int8_linear import quantize_per_token_int8

    x = _rows(m, k, m + k, dtype).to(cuda_device)
    codes, scale = quantize_per_token_int8(x)
    ref, ref_scale = _codes_of(x)
    assert codes.shape == x.shape and codes.stride(0) % 16 == 0
    assert np.array_equal(codes.cpu().numpy(), ref)
    assert (np.abs(scale.double().cpu().numpy() - ref_scale) <= ref_scale * 2.0 ** -24).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k", [(148, 1), (203, 323), (149, 1024), (301, 1025), (160, 8191), (150, 9001), (150, 3000),
                                 (150, 8192), (149, 16384), (148, 24576), (150, 24584), (148, 32768)])
def test_quantiser_of_many_rows(cuda_device, m, k, dtype):
    """As many rows as SMs and more: other numbers of threads a row, one row of them not finite."""
    from tilemix_b200.linear.int8_linear import quantize_per_token_int8

    x = _rows(m, k, m + k, dtype).to(cuda_device)
    if k % 3 == 0:  # a view: rows that start anywhere
        x = torch.nn.functional.pad(x, (1, 2))[:, 1:k + 1]
    ref, ref_scale = _codes_of(x)
    x[5, k // 2] = float("nan")
    x[6, k - 1] = float("-inf")
    codes, scale = quantize_per_token_int8(x)
    ref[5:7] = 0
    assert np.array_equal(codes.cpu().numpy(), ref)
    scale = scale.double().cpu().numpy()
    assert np.isnan(scale[5]) and np.isposinf(scale[6])
    fine = np.delete(np.arange(m), [5, 6])
    assert (np.abs(scale - ref_scale)[fine] <= ref_scale[fine] * 2.0 ** -24).all()


@pytest.mark.parametrize("m,n,k", [(1300, 4663, 323), (777, 93, 843), (100, 511, 2048), (260, 2449, 860), (90, 4097, 512)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_odd_output_rows(cuda_device, m, n, k, dtype):
    """Output rows that do not start on 16 bytes, and nothing written beside them."""
    from tilemix_b200._lib import TM_DTYPE_FP16, TM_DTYPE_FP32, launcher

    x8, xs, w8, ws = _operands(cuda_device, m, n, k, seed=m + n)
    out = torch.full((m + 2, n + 3), 7.0, dtype=dtype, device=cuda_device)
    inner = out[1:-1, 1:-2]
    launcher("tm_int8_matmul")(0, x8.data_ptr(), x8.stride(0), xs.data_ptr(), w8.data_ptr(), w8.stride(0), ws.data_ptr(),
                               0, inner.data_ptr(), inner.stride(0),
                               TM_DTYPE_FP16 if dtype == torch.float16 else TM_DTYPE_FP32, m, n, k)
    _check(inner, x8, xs, w8, ws)
    beside = out.clone()
    beside[1:-1, 1:-2] = 7
    assert (beside == 7).all()


def test_quantiser_takes_strided_and_unaligned_rows(cuda_device):
    from tilemix_b200.linear.int8_linear import quantize_per_token_int8

    wide = _rows(6, 500, 4, torch.float16).to(cuda_device)
    for x in (wide[:, 8:264], wide[:, 3:260], wide[::2, :256], wide[:, :1]):
        codes, _ = quantize_per_token_int8(x)
        assert np.array_equal(codes.cpu().numpy(), _codes_of(x)[0])


def test_quantiser_extremes(cuda_device):
    """The smallest and largest rows of bf16 and fp16, and rows that are not finite."""
    from tilemix_b200.linear.int8_linear import int8_linear, quantize_per_token_int8

    base = torch.tensor([1.0, -0.5, 0.25, 0.3, 0.9, -1.0, 0.0, 0.125])
    for dtype, sizes in ((torch.bfloat16, (1e-38, 3e38, 2.0 ** -120, 2.0 ** 100)), (torch.float16, (6e-5, 65000.0))):
        for size in sizes:
            x = (base * size).to(dtype)[None].to(cuda_device)
            assert np.array_equal(quantize_per_token_int8(x)[0].cpu().numpy(), _codes_of(x)[0]), (dtype, size)
    tiny = torch.tensor([[2.0 ** -133, -(2.0 ** -132), 0.0, 2.0 ** -131]]).to(torch.bfloat16).to(cuda_device)
    assert np.array_equal(quantize_per_token_int8(tiny)[0].cpu().numpy(), _codes_of(tiny)[0])
    x = torch.ones((4, 64), dtype=torch.float16, device=cuda_device)
    x[1, 5], x[2, 6] = float("inf"), float("nan")
    w8, ws = quantize_per_token_int8(torch.ones((32, 64), dtype=torch.float16, device=cuda_device))
    y = int8_linear(x, w8, ws)
    # 64 products of 1 * 1 in three roundings of the scales (fp32) and one of the result
    assert ((y[[0, 3]] - 64).abs() <= 64 * 2.0 ** -11).all() and y[1:3].isnan().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 200), (3, 5, 200), (0, 200), (2, 0, 200), (200,)])
def test_linear_layer(cuda_device, dtype, shape):
    from tilemix_b200.linear.int8_linear import Int8Linear, int8_matmul, quantize_per_token_int8

    torch.manual_seed(0)
    linear = torch.nn.Linear(200, 72).to(cuda_device, dtype)
    layer = Int8Linear(linear)
    assert layer.weight.shape == (72, 200) and layer.codes.stride(0) == 208
    x = torch.randn(shape, generator=torch.Generator().manual_seed(5)).to(cuda_device, dtype)
    y = layer(x)
    assert y.shape == shape[:-1] + (72,) and y.dtype == dtype
    flat = x.reshape(-1, 200)
    if flat.shape[0]:
        x8, xs = quantize_per_token_int8(flat)
        assert torch.equal(y.reshape(-1, 72), int8_matmul(x8, xs, layer.weight, layer.weight_scale, linear.bias.detach(),
                                                          out_dtype=dtype))
    assert torch.equal(layer(x.flip(-1).flip(-1)), y)
    with pytest.raises(TypeError):
        layer(x.float())


def test_refusals(cuda_device):
    from tilemix_b200.linear.int8_linear import int8_linear, int8_matmul, quantize_per_token_int8

    x8, xs, w8, ws = _operands(cuda_device, 4, 8, 64, seed=1)
    bad = [(ValueError, (x8[:, 4:36], xs, w8[:, :32], ws)), (ValueError, (x8, xs[:3], w8, ws)),
           (ValueError, (x8, xs, w8[:, :48], ws)), (TypeError, (x8.float(), xs, w8, ws)),
           (TypeError, (x8, xs.double(), w8, ws)), (ValueError, (x8.t()[:8], xs, w8, ws)),
           (TypeError, (x8, xs, w8, ws, torch.zeros(8, device=cuda_device))),
           (ValueError, (x8, xs, w8, ws, torch.zeros(7, dtype=torch.float16, device=cuda_device))),
           (RuntimeError, (x8.cpu(), xs, w8, ws)), (ValueError, (x8, xs, w8.cpu(), ws)),
           (ValueError, (torch.zeros((4, 60), dtype=torch.int8, device=cuda_device), xs, w8[:, :60], ws))]
    for exc, args in bad:
        with pytest.raises(exc):
            int8_matmul(*args)
    with pytest.raises(TypeError):
        int8_matmul(x8, xs, w8, ws, out_dtype=torch.int32)
    with pytest.raises(TypeError):
        int8_linear(torch.zeros((2, 64), device=cuda_device), w8, ws)
    with pytest.raises(ValueError):
        quantize_per_token_int8(torch.zeros((2, 0), dtype=torch.float16, device=cuda_device))
    k = 131072
    with pytest.raises(RuntimeError, match="status -4"):
        one = torch.zeros((1, k), dtype=torch.int8, device=cuda_device)
        int8_matmul(one, xs[:1], one, ws[:1])


def test_on_another_stream_and_in_graphs(cuda_device):
    """Captured, replayed with other inputs; two graphs at once on two streams."""
    from tilemix_b200.linear.int8_linear import int8_linear, quantize_per_token_int8

    g = torch.Generator().manual_seed(7)
    w8, ws = quantize_per_token_int8(torch.randn((1000, 2048), generator=g).to(cuda_device, torch.float16))
    feeds = [torch.randn((20, 2048), generator=g).to(cuda_device, torch.float16) for _ in range(4)]
    want = [int8_linear(x, w8, ws) for x in feeds]
    statics, graphs, outs = [torch.zeros_like(feeds[0]) for _ in range(2)], [], []
    for x in statics:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(int8_linear(x, w8, ws))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for i in range(0, 4, 2):
        for j, (st, graph) in enumerate(zip(streams, graphs)):
            with torch.cuda.stream(st):
                statics[j].copy_(feeds[i + j])
                graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[i]) and torch.equal(outs[1], want[i + 1])


@pytest.mark.parametrize("m,n", [(1, 40), (5, 1), (1, 1)])
@pytest.mark.parametrize("k", [100, 33, 4000])
def test_single_rows_need_no_padding(cuda_device, m, n, k):
    """The stride of a single row is never used: a contiguous one of any length is as good as a padded one."""
    from tilemix_b200.linear.int8_linear import int8_matmul

    x8, xs, w8, ws = _operands(cuda_device, m, n, k, seed=k)
    a, b = (t if t.shape[0] > 1 else t[0].clone()[None] for t in (x8, w8))
    assert m > 1 or a.stride(0) == k
    assert n > 1 or b.stride(0) == k
    _check(int8_matmul(a, xs, b, ws), x8, xs, w8, ws)


def test_a_layer_keeps_its_scales_through_conversions(cuda_device):
    """half(), bfloat16() and moves change the type of the activations and of the bias; codes and scales stay as they are."""
    from tilemix_b200.linear.int8_linear import Int8Linear, int8_linear

    torch.manual_seed(0)
    layer = Int8Linear(torch.nn.Linear(200, 72).to(cuda_device, torch.float16))
    codes, scale, bias = layer.codes.clone(), layer.weight_scale.clone(), layer.bias.clone()
    x = torch.randn((6, 200), generator=torch.Generator().manual_seed(1)).to(cuda_device)
    for convert, dtype in ((lambda m: m.half(), torch.float16), (lambda m: m.to(torch.bfloat16), torch.bfloat16),
                           (lambda m: m.cpu().to(cuda_device), torch.bfloat16)):
        layer = convert(layer)
        assert torch.equal(layer.codes, codes) and torch.equal(layer.weight_scale, scale)
        assert layer.dtype == layer.bias.dtype == dtype
        want = int8_linear(x.to(dtype), codes[:, :200], scale, bias.to(dtype))
        assert torch.equal(layer(x.to(dtype)), want)
    with pytest.raises(TypeError):
        layer(x.half())
    layer = layer.float()
    assert torch.equal(layer.weight_scale, scale)
    with pytest.raises(TypeError):
        layer(x)


def test_a_layer_made_in_inference_mode(cuda_device):
    """Its codes are laid out as those of any other layer: rows on 16 bytes, also after a move."""
    from tilemix_b200.linear.int8_linear import Int8Linear

    torch.manual_seed(0)
    linear = torch.nn.Linear(200, 72).to(cuda_device, torch.float16)
    x = torch.randn((3, 200), generator=torch.Generator().manual_seed(1)).half().to(cuda_device)
    with torch.inference_mode():
        layer = Int8Linear(linear)
        assert layer.codes.shape == (72, 208)
        want = layer(x)
        assert torch.equal(layer.cpu().to(cuda_device)(x), want)
    other = Int8Linear(linear)
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), want)


# Sizes that reach every form of the product: weights on the lanes with 16, 32 and 64 tokens a tile, tokens on the lanes with
# 64, 128 and 256 channels, pairs of SMs with 128 to 256 channels, K whole and in 2, 4 and 8 parts; many tiles a CTA
# and more steps than the ring has stages.
FORMS = [(2, 4162, 2216), (13, 3253, 1974), (5, 2110, 4506), (3, 45001, 1111), (28, 38, 1832), (30, 2054, 4667),
         (20, 45001, 1111), (49, 11854, 3358), (43, 7067, 11986), (60, 3584, 18944), (42, 1030, 8102), (50, 45001, 1011),
         (131, 10668, 104), (302, 1435, 3385), (278, 655, 3194), (367, 2498, 9553), (37, 43396, 641), (263, 31780, 132),
         (1813, 7269, 530), (246, 8453, 13615), (4182, 2147, 1078), (700, 7755, 2841), (4155, 2066, 1100),
         (1435, 6284, 782), (3935, 2516, 780), (777, 4608, 3584), (3336, 3455, 822)]


@pytest.mark.parametrize("m,n,k", FORMS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_every_form_matches_exact_sums(cuda_device, m, n, k, dtype):
    from tilemix_b200.linear.int8_linear import int8_matmul

    x8, xs, w8, ws = _operands(cuda_device, m, n, k, seed=m + n + k)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(1)).to(cuda_device, dtype)
    out = int8_matmul(x8, xs, w8, ws, bias, out_dtype=dtype)
    _check(out, x8, xs, w8, ws, bias)
    for _ in range(3):
        assert torch.equal(int8_matmul(x8, xs, w8, ws, bias, out_dtype=dtype), out)


@pytest.mark.parametrize("m,n,k", [(3935, 2516, 780), (2000, 3000, 18944)])
def test_a_token_does_not_depend_on_its_batch_in_the_large_forms(cuda_device, m, n, k):
    from tilemix_b200.linear.int8_linear import int8_matmul

    x8, xs, w8, ws = _operands(cuda_device, m, n, k, seed=5)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(2)).to(cuda_device, torch.bfloat16)
    full = int8_matmul(x8, xs, w8, ws, bias, out_dtype=torch.bfloat16)
    for part in (3, 30, 50, 90, 200, 600, 777, 1500, m - 1):
        assert torch.equal(int8_matmul(x8[:part], xs[:part], w8, ws, bias, out_dtype=torch.bfloat16), full[:part]), part


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 3, 8])
@pytest.mark.parametrize("m,k", [(148, 2056), (160, 4096), (149, 8200), (151, 12288), (148, 16400), (150, 24576)])
def test_quantiser_of_many_wide_rows(cuda_device, m, k, offset, dtype):
    """Rows on 16 bytes, and views that start elsewhere."""
    from tilemix_b200.linear.int8_linear import quantize_per_token_int8

    x = torch.nn.functional.pad(_rows(m, k, m + k, dtype), (offset, 8 - offset)).to(cuda_device)[:, offset:offset + k]
    ref, ref_scale = _codes_of(x)
    x[5, k // 2], x[6, k - 1] = float("nan"), float("-inf")
    ref[5:7] = 0
    codes, scale = quantize_per_token_int8(x)
    assert np.array_equal(codes.cpu().numpy(), ref)
    scale = scale.double().cpu().numpy()
    assert np.isnan(scale[5]) and np.isposinf(scale[6])
    fine = np.delete(np.arange(m), [5, 6])
    assert (np.abs(scale - ref_scale)[fine] <= ref_scale[fine] * 2.0 ** -24).all()


def test_more_than_32_bits_of_elements(cuda_device):
    """Inputs and outputs of over 2^31 elements: the last rows are those of a small call."""
    from tilemix_b200.linear.int8_linear import int8_matmul, quantize_per_token_int8

    m, n, k = 70001, 40008, 96
    x8, xs, w8, ws = _operands(cuda_device, m, n, k, seed=3)
    out = int8_matmul(x8, xs, w8, ws)
    assert out.numel() > 2**31
    for rows in (slice(0, 40), slice(2**31 // n - 20, 2**31 // n + 20), slice(m - 40, m)):
        assert torch.equal(out[rows], int8_matmul(x8[rows], xs[rows], w8, ws))
    codes, scale = quantize_per_token_int8(out)
    odd, odd_scale = quantize_per_token_int8(out[:, :8001])
    for rows in (slice(0, 40), slice(2**31 // n - 20, 2**31 // n + 20), slice(m - 40, m)):
        few, few_scale = quantize_per_token_int8(out[rows])
        assert torch.equal(codes[rows], few) and torch.equal(scale[rows], few_scale)
        few, few_scale = quantize_per_token_int8(out[rows, :8001])
        assert torch.equal(odd[rows], few) and torch.equal(odd_scale[rows], few_scale)
