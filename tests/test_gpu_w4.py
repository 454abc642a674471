"""4-bit weights on the GPU against plain float64 restatements: quantising and
restoring bit for bit, products within the rounding of fp32 sums."""

import math

import pytest
import torch
import torch.nn as nn

from conftest import announce, load_pkg

pytestmark = pytest.mark.gpu
pkg = load_pkg()
w4 = pkg.w4
MAGNITUDES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
GROUPS = (32, 64, 128)


def ref_quantize(w, group):
    """Scales [out, groups] (fp32 of bf16) and codes [out, in padded to 128], on the CPU."""
    out, d_in = w.shape
    w = torch.nn.functional.pad(w.float().cpu(), (0, -d_in % 128)).view(out, -1, group)
    top = w.abs().amax(2)
    scale = (top * (1.0 / 6.0)).to(torch.bfloat16).float()
    limit = torch.finfo(torch.float32).max / 6                         # of a scale whose weights fp32 holds
    scale = torch.where(scale > limit, torch.tensor(0x7e2a, dtype=torch.int16).view(torch.bfloat16).float(), scale)
    bad = ~torch.isfinite(w).all(2)
    scale[bad] = math.nan
    s, a = scale.double().unsqueeze(2), w.abs().double()
    ratio = torch.where(s > 0, a / s, torch.zeros_like(a)).clamp(max=7.0)
    dist = (ratio.unsqueeze(3) - MAGNITUDES).abs()
    # nearest; of two equally near the one with an even mantissa bit (an even code)
    near = dist == dist.min(3, keepdim=True).values
    even = near & (torch.arange(8) % 2 == 0)
    pick = torch.where(even.any(3, keepdim=True), even, near)
    code = pick.int().argmax(3)
    code[~(s > 0).expand_as(code)] = 0
    code = torch.where((w < 0) & (code > 0), code + 8, code)
    return scale, code.reshape(out, -1)


def ref_values(scale, code, d_in):
    out = code.shape[0]
    v = MAGNITUDES[code & 7] * torch.where(code > 7, -1.0, 1.0)
    return (v.view(out, scale.shape[1], -1) * scale.double().unsqueeze(2)).view(out, -1)[:, :d_in]


def ref_pack(code):
    """include/rwkv_w4.h's layout, byte by byte."""
    out, d_in = code.shape
    n, k = -(-out // 16), d_in // 128
    full = torch.zeros(16 * n, d_in, dtype=torch.int64)
    full[:out] = code
    N, K, g, r, j, b = (torch.arange(x).view([-1 if i == a else 1 for i in range(6)])
                        for a, x in enumerate((n, k, 4, 16, 4, 4)))
    low = full[16 * N + r, 128 * K + 32 * j + 8 * g + 2 * b]
    high = full[16 * N + r, 128 * K + 32 * j + 8 * g + 2 * b + 1]
    return (low | high << 4).view(n, k, 4, 16, 16).to(torch.uint8)


def rand(*shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1), (16, 128), (17, 129), (5, 4), (33, 96), (129, 1000), (256, 768), (40, 72)])
def test_quantize_and_restore(shape, dtype, group):
    announce("w4 quantize", shape, dtype, group)
    w = rand(*shape, seed=1, dtype=dtype, scale=0.02)
    q = w4.quantize(w, group)
    scale, code = ref_quantize(w, group)
    assert torch.equal(q.packed.cpu(), ref_pack(code))
    n, k = q.packed.shape[:2]
    got = q.scales.cpu().float().transpose(1, 2).reshape(16 * n, -1)
    assert torch.equal(got[:shape[0]], scale) and not got[shape[0]:].any()
    want = ref_values(scale, code, shape[1])
    assert torch.equal(w4.dequantize(q).cpu().double(), want)          # exact in fp32
    assert torch.equal(w4.dequantize(q, torch.bfloat16).cpu(), want.float().to(torch.bfloat16))


def test_quantize_edges():
    """Midpoints, saturation, signed zeros, empty and denormal groups, infinities and NaN."""
    announce("w4 quantize edges")
    w = torch.zeros(8, 64)
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    w[0, :7], w[0, 7:14], w[0, 20] = mids, -mids, 6.0                  # scale exactly 1
    w[1, :14] = torch.nextafter(torch.cat([mids, mids]), torch.tensor([9.0] * 7 + [0.0] * 7))
    w[1, 20] = -6.0
    w[2, 3] = -0.0
    w[3, :4] = torch.tensor([1e-38, -1e-39, 1e-45, 3e-39])
    w[4, 1], w[4, 40] = math.inf, 1.0
    w[5, 33], w[5, 2] = math.nan, 1.0
    w[6, 0], w[6, 1] = 3.4e38, -1e38
    w[7, 0] = 1e-45                                                     # its scale rounds to zero
    q = w4.quantize(w.cuda(), 32)
    scale, code = ref_quantize(w, 32)
    assert torch.equal(q.packed.cpu(), ref_pack(code))
    got, want = w4.dequantize(q).cpu().double(), ref_values(scale, code, 64)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(), want.nan_to_num())
    assert got[4, :32].isnan().all() and got[4, 40] == 6 * float(torch.tensor(1 / 6).bfloat16()) and got[5, 33:].isnan().all()
    assert got[0, :7].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0]
    assert got[1, :7].tolist() == [0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    assert got[1, 7:14].tolist() == [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0]


def check_linear(x, q, d_out, d_in, on="cpu"):
    """Against float64 products of the same values. A sum of K products in fp32,
    in any order and however a matrix instruction rounds inside (one unit in the
    last place, 2^-23, for each addition), is off by at most (K + 8) 2^-23 sum
    |x w|; fp32 parts lose 2^-23 |x w| more; the result is rounded once."""
    y = w4.linear(x, q)
    assert y.dtype == x.dtype and y.shape == (*x.shape[:-1], d_out)
    w = w4.dequantize(q).to(on).double()
    xd = x.to(on).double()
    want, mass = xd @ w.t(), xd.abs() @ w.abs().t()
    last = 2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -23
    err = (y.to(on).double() - want).abs()
    bound = (d_in + 9) * 2.0 ** -23 * mass + last * want.abs() + 1e-37
    assert (err <= bound).all(), float((err / bound).max())
    # and as a whole far nearer than that bound
    rel = float(err.norm() / want.norm().clamp(min=1e-300))
    assert rel <= (2.0 ** -8 if x.dtype == torch.bfloat16 else 2e-6), rel


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,d_out,d_in,group", [
    (1, 16, 128, 32), (1, 1, 1, 64), (1, 768, 768, 64), (2, 100, 300, 128), (3, 777, 1000, 32),
    (7, 64, 64, 64), (8, 48, 1024, 128), (16, 33, 129, 64), (17, 256, 768, 128), (31, 80, 416, 32),
    (33, 130, 2048, 64), (64, 512, 256, 32), (65, 96, 640, 64), (100, 300, 333, 128),
    (129, 128, 512, 64), (257, 200, 1152, 32), (300, 1000, 200, 128), (1, 40, 9000, 64)])
def test_linear(rows, d_out, d_in, group, dtype):
    announce("w4 linear", rows, d_out, d_in, group, dtype)
    q = w4.quantize(rand(d_out, d_in, seed=2, scale=0.05), group)
    check_linear(rand(rows, d_in, seed=3, dtype=dtype), q, d_out, d_in)


@pytest.mark.parametrize("dtype,rows,d_out,d_in,group", [
    # up to 16 rows with one, two and four tiles of outputs a workgroup; up to 64 without a share
    (torch.bfloat16, 5, 8200, 140, 64), (torch.bfloat16, 3, 32800, 130, 128), (torch.float32, 9, 8200, 140, 32),
    (torch.float32, 2, 32800, 130, 64), (torch.bfloat16, 18, 8523, 131, 32), (torch.float32, 17, 8828, 543, 64),
    (torch.float32, 33, 16, 429, 128),
    # each tile, with an odd and an even number of blocks of inputs, one workgroup a tile or several
    (torch.bfloat16, 66, 16, 130, 64), (torch.bfloat16, 40, 17, 1256, 128), (torch.bfloat16, 165, 16, 5510, 32),
    (torch.bfloat16, 65, 18481, 132, 32), (torch.bfloat16, 96, 20443, 128, 64), (torch.bfloat16, 18, 8851, 3844, 64),
    (torch.bfloat16, 33, 24702, 137, 128), (torch.bfloat16, 52, 25785, 128, 32), (torch.bfloat16, 34, 2906, 4608, 64),
    (torch.bfloat16, 264, 25527, 130, 64), (torch.bfloat16, 339, 28674, 128, 128), (torch.bfloat16, 339, 28671, 256, 32),
    (torch.float32, 1474, 32, 648, 64), (torch.float32, 34, 8474, 133, 128), (torch.float32, 19, 23877, 128, 32),
    (torch.float32, 162, 67, 5532, 32), (torch.float32, 69, 67, 5683, 64), (torch.float32, 17, 33985, 129, 64),
    (torch.float32, 20, 34947, 128, 128), (torch.float32, 1064, 129, 1325, 128), (torch.float32, 33, 333, 5426, 32)])
def test_linear_every_form(dtype, rows, d_out, d_in, group):
    announce("w4 linear form", dtype, rows, d_out, d_in, group)
    q = w4.quantize(rand(d_out, d_in, seed=31, scale=0.05), group)
    check_linear(rand(rows, d_in, seed=32, dtype=dtype), q, d_out, d_in, on="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 20, 200])
def test_linear_hears_every_element(rows, dtype):
    """One activation at a time: the outputs are the weights of its input, exactly."""
    announce("w4 linear one-hot", rows, dtype)
    d_out, d_in = 50, 200
    q = w4.quantize(rand(d_out, d_in, seed=4), 32)
    w = w4.dequantize(q, dtype)
    for k0 in range(0, d_in, rows):
        ks = torch.arange(k0, k0 + rows, device="cuda") % d_in
        x = torch.zeros(rows, d_in, device="cuda", dtype=dtype)
        x[torch.arange(rows), ks] = 1.0
        assert torch.equal(w4.linear(x, q), w.t()[ks])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 19, 150])
@pytest.mark.parametrize("d_in", [256, 203])
def test_linear_infinities_and_nan_stay_in_their_rows(rows, d_in, dtype):
    announce("w4 linear non-finite", rows, d_in, dtype)
    d_out = 70
    q = w4.quantize(rand(d_out, d_in, seed=5), 64)
    w = w4.dequantize(q).cpu().double()
    x = rand(rows, d_in, seed=6, dtype=dtype)
    x[0, 3] = math.inf
    if rows > 1:
        x[1, 5], x[1, 9], x[2, 7], x[3, d_in - 1] = math.inf, -math.inf, math.nan, -math.inf
        x[4, 0] = torch.finfo(dtype).max
    y, want = w4.linear(x, q).cpu().double(), x.cpu().double() @ w.t()
    assert torch.equal(y.isnan(), want.isnan())
    assert torch.equal(y == math.inf, want.to(dtype) == math.inf)
    assert torch.equal(y == -math.inf, want.to(dtype) == -math.inf)
    fine = y.isfinite()
    assert torch.allclose(y[fine], want[fine], rtol=2.0 ** -7, atol=1e-3)


def test_a_nan_group_reaches_its_output_only():
    announce("w4 linear NaN weight")
    w = rand(40, 300, seed=7)
    w[11, 170] = math.nan
    q = w4.quantize(w, 64)
    y = w4.linear(rand(3, 300, seed=8), q)
    assert y[:, 11].isnan().all() and y.isnan().sum() == 3


def test_fp32_activations_of_every_size():
    """x is cut into three bf16 parts: nothing is lost from 2^-100 to 2^120."""
    announce("w4 linear fp32 range")
    q = w4.quantize(torch.eye(64, device="cuda") * 6.0, 32)          # 6 on the diagonal, scale 1
    x = rand(1, 64, seed=9) * torch.exp2(torch.linspace(-100, 120, 64, device="cuda"))
    y = w4.linear(x, q)
    assert torch.allclose(y, 6.0 * x, rtol=2.0 ** -22, atol=0.0)


def test_linear_results_do_not_depend_on_the_call():
    """The same row, alone and among others of the same launch, again and again."""
    announce("w4 linear repeat")
    q = w4.quantize(rand(512, 768, seed=10), 64)
    x = rand(13, 768, seed=11, dtype=torch.bfloat16)
    y = w4.linear(x, q)
    for _ in range(3):
        assert torch.equal(w4.linear(x, q), y)
    assert torch.equal(w4.linear(x[4:5], q), y[4:5])


def test_linear_shapes_strides_and_empty_calls():
    announce("w4 linear shapes")
    q = w4.quantize(rand(24, 136, seed=12), 64)
    x = rand(2, 3, 136, seed=13, dtype=torch.bfloat16)
    y = w4.linear(x, q)
    assert y.shape == (2, 3, 24) and torch.equal(y.view(6, 24), w4.linear(x.view(6, 136), q))
    assert torch.equal(w4.linear(x[:, -1], q), y[:, -1])                       # strided rows
    wide = rand(3, 272, seed=14, dtype=torch.bfloat16)
    assert torch.equal(w4.linear(wide[:, ::2], q), w4.linear(wide[:, ::2].contiguous(), q))
    flat = rand(137, seed=15, dtype=torch.bfloat16)
    assert torch.equal(w4.linear(flat[1:], q), w4.linear(flat[1:].clone(), q))  # begins anywhere
    assert w4.linear(x[:0], q).shape == (0, 3, 24)
    w = rand(24 * 136 + 1, seed=16)[1:].view(24, 136)
    assert torch.equal(w4.quantize(w).packed, w4.quantize(w.clone()).packed)
    wt = rand(136, 24, seed=17).t()
    assert torch.equal(w4.quantize(wt).packed, w4.quantize(wt.contiguous()).packed)


def test_linear_on_another_stream_and_in_a_graph():
    announce("w4 linear stream and graph")
    q = w4.quantize(rand(256, 512, seed=18), 128)
    xs = [rand(4, 512, seed=19 + i, dtype=torch.bfloat16) for i in range(3)]
    want = [w4.linear(x, q) for x in xs]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = w4.linear(xs[0], q)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want[0])
    held = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = w4.linear(held, q)
    for x, w in zip(xs + xs, want + want):
        held.copy_(x)
        graph.replay()
        assert torch.equal(out, w)
        torch.cuda.synchronize()


def test_refusals():
    announce("w4 refusals")
    q = w4.quantize(rand(24, 136, seed=20), 64)
    x = rand(2, 136, seed=21)
    for bad, exc in [(lambda: w4.quantize(x, 48), ValueError), (lambda: w4.quantize(x.cpu()), ValueError),
                     (lambda: w4.quantize(x[0]), ValueError), (lambda: w4.quantize(x.half()), TypeError),
                     (lambda: w4.quantize(x[:0]), ValueError), (lambda: w4.linear(x.half(), q), TypeError),
                     (lambda: w4.linear(x[:, 1:], q), ValueError), (lambda: w4.linear(x.cpu(), q), ValueError),
                     (lambda: w4.linear(x.clone().requires_grad_(), q), RuntimeError),
                     (lambda: w4.dequantize(q, torch.float16), TypeError),
                     (lambda: w4.W4Weight(q.packed, q.scales, 24, 136, 32), ValueError),
                     (lambda: w4.W4Weight(q.packed[:1], q.scales, 24, 136, 64), ValueError),
                     (lambda: w4.W4Weight(q.packed.int(), q.scales, 24, 136, 64), ValueError),
                     (lambda: w4.W4Weight(q.packed, q.scales.cpu(), 24, 136, 64), ValueError),
                     (lambda: w4.W4Linear.from_linear(nn.Linear(8, 8).cuda()), ValueError)]:
        with pytest.raises(exc):
            bad()
    with torch.no_grad():
        w4.linear(x.clone().requires_grad_(), q)


def test_module_and_model():
    announce("w4 module")
    lin = nn.Linear(192, 80, bias=False).cuda()
    mod = w4.W4Linear.from_linear(lin, 32)
    x = rand(5, 192, seed=22)
    with torch.no_grad():
        assert torch.equal(mod(x), w4.linear(x, w4.quantize(lin.weight, 32)))
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = mod(x)
        assert y.dtype == torch.bfloat16 and torch.equal(y, w4.linear(x.bfloat16(), mod.weight))
    again = w4.W4Linear(w4.quantize(torch.zeros(80, 192, device="cuda"), 32))
    again.load_state_dict(mod.state_dict())
    with torch.no_grad():
        assert torch.equal(again(x), mod(x))
    model = pkg.model.AutoRegressiveModel(100, 2, 128, 2).init_random().cuda()
    w4.quantize_model(model, 64)
    kinds = [type(m) for m in model.modules()]
    assert kinds.count(w4.W4Linear) == 2 * 6 + 1 and nn.Linear not in kinds


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 20, 100])
def test_sums_overflow_only_where_the_result_does(rows, dtype, group):
    """Activations near the largest number, weights so small that the results are
    ordinary: a group's sum before its scale, and the sum of some groups, are not."""
    announce("w4 linear near the largest number", rows, dtype, group)
    d_out, d_in = 40, 512
    small = w4.quantize(torch.full((d_out, d_in), 1e-3, device="cuda"), group)
    check_linear(torch.full((rows, d_in), 3e38, device="cuda", dtype=dtype), small, d_out, d_in)
    two = torch.zeros(rows, d_in, device="cuda", dtype=dtype)
    two[:, :2] = 3e38
    check_linear(two, w4.quantize(torch.full((d_out, d_in), 0.06, device="cuda"), group), d_out, d_in)
    # 256 inputs of either sign: the sum is 0, that of the first half 256 * 0.1 * 3e38;
    # check_linear's bound on the rounding of sums
    x = torch.full((rows, d_in), 3e38, device="cuda", dtype=dtype)
    x[:, d_in // 2:] = -3e38
    y = w4.linear(x, w4.quantize(torch.full((d_out, d_in), 0.1, device="cuda"), group))
    assert float(y.double().abs().max()) <= (d_in + 9) * 2.0 ** -23 * d_in * 0.101 * 3e38


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 20, 100])
def test_the_smallest_activations(rows, dtype):
    """Scale 1, one activation a row and weight: bf16 ones are exact down to 2^-133,
    fp32 ones lose what is below that, and a result is a multiple of 2^-139."""
    announce("w4 linear near the smallest number", rows, dtype)
    w = torch.zeros(16, 64)
    w[:, :8] = MAGNITUDES.float()
    w[:, 40] = 6.0                                                     # of the other group
    q = w4.quantize(w.cuda(), 32)
    g = torch.Generator().manual_seed(33)
    for power in range(-149, -90):
        x = torch.zeros(rows, 64, dtype=torch.float64)
        x[torch.arange(rows), torch.arange(rows) % 8] = torch.exp2(torch.rand(rows, generator=g, dtype=torch.float64) + power)
        x = x.to(dtype)
        y = w4.linear(x.cuda(), q).cpu().double()
        want = x.double() @ w.double().t()
        if dtype == torch.bfloat16:
            assert torch.equal(y, want.to(dtype).double()), power
        else:
            assert ((y - want).abs() <= 6 * 2.0 ** -133 + 2.0 ** -139 + 2.0 ** -23 * want.abs()).all(), power


def test_forward_mode_is_refused():
    """A result without a tangent would be read as a constant."""
    announce("w4 linear, forward mode")
    fw = torch.autograd.forward_ad
    q = w4.quantize(rand(24, 136, seed=34), 64)
    mod = w4.W4Linear(q)
    x = rand(2, 136, seed=35)
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        for call in (lambda z: w4.linear(z, q), mod):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                    call(dual)
        with torch.autocast("cuda", dtype=torch.bfloat16), pytest.raises(NotImplementedError):
            mod(dual)
        want = w4.linear(x, q)                                # no tangent: nothing is lost
    assert torch.equal(w4.linear(x, q), want)


@pytest.mark.parametrize("dtype,rows,d_out,d_in,group", [
    # five blocks of inputs a workgroup and more, in which LDS and the registers ahead
    # are used again: an odd and an even number, the inputs shared or not, the last
    # share as long or shorter, inputs of whole blocks and not
    (torch.bfloat16, 231, 28672, 640, 64), (torch.bfloat16, 257, 25705, 658, 32), (torch.bfloat16, 2048, 4096, 700, 128),
    (torch.bfloat16, 34, 16924, 4480, 128), (torch.bfloat16, 33, 16971, 4351, 64), (torch.bfloat16, 36, 16414, 5252, 32),
    (torch.bfloat16, 33, 16499, 5248, 64), (torch.bfloat16, 35, 26025, 640, 128), (torch.bfloat16, 33, 27730, 642, 32),
    (torch.bfloat16, 33, 3531, 4736, 64), (torch.bfloat16, 34, 2691, 7379, 128), (torch.bfloat16, 65, 19285, 520, 64),
    (torch.bfloat16, 17, 8346, 4096, 32), (torch.bfloat16, 17, 5475, 7300, 128), (torch.bfloat16, 1930, 22, 2827, 64),
    (torch.float32, 38, 16591, 640, 64), (torch.float32, 36, 17074, 658, 128), (torch.float32, 33, 1315, 11285, 32),
    (torch.float32, 33, 8215, 2048, 128), (torch.float32, 35, 1539, 9600, 64), (torch.float32, 33, 8406, 2204, 32),
    (torch.float32, 33, 8654, 533, 32), (torch.float32, 34, 8518, 768, 64), (torch.float32, 609, 66, 6413, 128),
    (torch.float32, 566, 67, 9088, 64), (torch.float32, 489, 65, 8320, 32), (torch.float32, 478, 296, 2069, 64),
    (torch.float32, 1770, 43, 640, 128)])
def test_linear_tiles_of_many_blocks(dtype, rows, d_out, d_in, group):
    announce("w4 linear tiles", dtype, rows, d_out, d_in, group)
    q = w4.quantize(rand(d_out, d_in, seed=41, scale=0.05), group)
    check_linear(rand(rows, d_in, seed=42, dtype=dtype), q, d_out, d_in, on="cuda")


@pytest.mark.parametrize("dtype,rows,d_out,d_in", [(torch.bfloat16, 575, 17, 7434), (torch.bfloat16, 33, 3531, 4736),
                                                   (torch.float32, 361, 16, 11520)])
def test_shared_inputs_on_two_streams_and_in_a_graph(dtype, rows, d_out, d_in):
    """Products with a workspace: two streams at a time do not share it, and a graph keeps its own."""
    announce("w4 linear with a workspace, streams and graph", dtype, rows, d_out, d_in)
    native = pkg._native
    code = native.DTYPE_BF16 if dtype == torch.bfloat16 else native.DTYPE_F32
    assert native.lib().rwkv_w4_linear_workspace_bytes(rows, d_out, d_in, code) > 0
    q = w4.quantize(rand(d_out, d_in, seed=43), 64)
    xs = [rand(rows, d_in, seed=44 + i, dtype=dtype) for i in range(3)]
    want = [w4.linear(x, q) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(8):
        for s, x, out in zip(streams, xs, got):
            with torch.cuda.stream(s):
                out.append(w4.linear(x, q))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for out, w in zip(got, want):
        assert all(torch.equal(y, w) for y in out)
    held = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = w4.linear(held, q)
    for x, w in zip(xs + xs, want + want):
        held.copy_(x)
        assert torch.equal(w4.linear(x, q), w)                        # eager work between the replays
        graph.replay()
        assert torch.equal(out, w)
        torch.cuda.synchronize()
