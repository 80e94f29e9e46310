"""4-bit storage and its products against float64.

Quantisation is compared bit for bit: every step of it is exact but the one rounding.  Products: the products of the 4-bit
values are exact and each of the cols additions in fp32 is off by at most one step (2^-23) of a partial sum that is at most
sum |a b|; the result is then rounded once to its type (half a step, eps / 2, and in fp16 half a subnormal step, 2^-25)."""
import math

import pytest
import torch

from oracle import teacher_oracle as to

FP = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def features(rows, cols, dt, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(cols, generator=g))).to(dt)


def bound(terms, mass, want, dt):
    """mass = sum |a b| of every output"""
    return (terms + 8) * 2.0 ** -23 * mass + torch.finfo(dt).eps / 2 * want.abs() * (1 + 1e-6) + TINY[dt]


# ---- CPU: the oracle on cases checked by hand, refusals --------------------------------------------------------------
def test_oracle_by_hand():
    x = torch.zeros(1, 64)
    x[0, :9] = torch.tensor([7.9, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.01])   # scale 1: floor(log2 7.9) = 2
    x[0, 32] = 2.0 ** -140
    v, code = to.mx4_round(x)
    assert code.tolist() == [[127, 0]]
    assert v[0, :9].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -6.0]
    assert float(v[0, 32]) == 0.0                                                  # 2^-13 of the smallest scale 2^-127
    codes, scales = to.mx4_pack(x)
    assert codes.shape == (1, 1, 128) and codes[0, 0, :5].tolist() == [0x07, 0x22, 0x44, 0x66, 0x0F]
    assert scales[0, 0, :2].tolist() == [127, 0]


def test_refusals_without_a_gpu():
    from msf_wsi_amd import _lib, quant

    with pytest.raises(_lib.MsfwsiHipError):
        quant.quantize_mx4(torch.zeros(2, 32))
    with pytest.raises(_lib.MsfwsiHipError):
        quant.MX4Tensor(torch.zeros(1, 2, 128, dtype=torch.uint8), torch.zeros(1, 2, 8, dtype=torch.uint8), 32)
    with pytest.raises(TypeError):
        quant.mx4_linear(torch.zeros(2, 32), torch.zeros(3, 32))


def test_c_entry_checks(hip_lib):
    """bad sizes come back as an error code before anything is launched"""
    assert hip_lib.msfwsi_mx4_quantize(7, None, 32, 1, 32, None, None, None) == -1
    assert hip_lib.msfwsi_mx4_quantize(0, None, 32, 1, 32, None, None, None) == -1     # no memory
    assert hip_lib.msfwsi_mx4_quantize(0, None, 16, 2, 32, None, None, None) == -1     # rows overlap
    assert hip_lib.msfwsi_mx4_quantize(0, None, 32, 0, 32, None, None, None) == 0      # no rows
    assert hip_lib.msfwsi_mx4_dequantize(0, None, None, 1, 0, None, None) == -1
    assert hip_lib.msfwsi_mx4_dgrad(0, None, 4, 1, None, None, 0, 32, 0, None, None, None) == -1


# ---- GPU -------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 256), (3, 31), (7, 33), (9, 255), (5, 257), (130, 1001), (64, 2048), (17, 4608)])
def test_quantize_bit_for_bit(hip_lib, dt, rows, cols):
    from msf_wsi_amd import quant

    x = features(rows, cols, FP[dt], rows * 7919 + cols)
    codes, scales = to.mx4_pack(x)
    q = quant.quantize_mx4(x.cuda())
    assert torch.equal(q.scales.cpu(), scales)
    assert torch.equal(q.codes.cpu(), codes)
    v, _ = to.mx4_round(x)
    assert torch.equal(q.dequantize().cpu().double(), v)
    assert torch.equal(q.dequantize(torch.bfloat16).cpu(), v.to(torch.bfloat16))


@pytest.mark.gpu
def test_quantize_every_border_and_scale(hip_lib):
    """all midpoints and their neighbours under every scale an fp32 block can take, subnormal blocks among them"""
    from msf_wsi_amd import quant

    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0])
    line = torch.cat([mids, torch.nextafter(mids, torch.tensor(0.0)), torch.nextafter(mids, torch.tensor(9.0))])
    block = torch.zeros(32)
    block[:27], block[27:31], block[31] = line, torch.tensor([4.0, 0.0, -0.5, 1e-3]), -7.5
    rows = []
    for e in range(-149, 126):
        rows.append(torch.ldexp(block.double(), torch.tensor(e)).float())
    x = torch.stack(rows)
    q = quant.quantize_mx4(x.cuda())
    codes, scales = to.mx4_pack(x)
    assert torch.equal(q.scales.cpu(), scales) and torch.equal(q.codes.cpu(), codes)
    assert torch.equal(q.dequantize().cpu().double(), to.mx4_round(x)[0])


@pytest.mark.gpu
def test_quantize_nonfinite_and_empty(hip_lib):
    from msf_wsi_amd import quant

    x = torch.ones(4, 96)
    x[0, 5], x[1, 40], x[2, 95] = math.nan, math.inf, -math.inf
    x[3] = 0.0
    q = quant.quantize_mx4(x.cuda())
    assert q.scales[0, :, :3].tolist() == [[255, 125, 125], [125, 255, 125], [125, 125, 255], [0, 0, 0]]
    back = q.dequantize().cpu()
    assert back[0, :32].isnan().all() and back[1, 32:64].isnan().all() and back[2, 64:].isnan().all()
    assert int(back.isnan().sum()) == 96 and float(back[3].abs().max()) == 0.0
    none = quant.quantize_mx4(torch.zeros(0, 40, device="cuda"))
    assert none.shape == (0, 40) and none.dequantize().shape == (0, 40)
    w = quant.quantize_mx4(x[3:].cuda())
    assert quant.mx4_linear(torch.zeros(0, 96, device="cuda"), w).shape == (0, 1)
    y = quant.mx4_linear(x.cuda(), quant.quantize_mx4(torch.ones(2, 96, device="cuda"))).cpu()
    assert y[:3].isnan().all() and y[3].tolist() == [0.0, 0.0]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
@pytest.mark.parametrize("offset,pitch", [(0, 300), (1, 301), (3, 517)])
def test_quantize_slices(hip_lib, dt, offset, pitch):
    """rows of a wider tensor at any alignment: the same codes as of a copy"""
    from msf_wsi_amd import quant

    base = features(11, pitch + 8, FP[dt], pitch).cuda()
    part = base[:, offset:offset + 291]
    a, b = quant.quantize_mx4(part), quant.quantize_mx4(part.contiguous())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    t = base[:, :11].t()
    assert torch.equal(quant.quantize_mx4(t).codes, quant.quantize_mx4(t.contiguous()).codes)


SIZES = [(1, 1, 1), (1, 256, 1000), (2, 513, 33), (5, 64, 7), (31, 255, 65), (33, 1001, 129), (64, 2048, 512), (130, 300, 257), (257, 4608, 300),
         (300, 256, 1), (1, 18432, 40), (16, 9216, 64), (520, 2304, 391), (4096, 300, 4100), (40, 18432, 70), (33, 70, 3000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear_forward_and_gradient(hip_lib, dt, M, K, N):
    from msf_wsi_amd import quant

    dt = FP[dt]
    g = torch.Generator().manual_seed(M * 31 + K * 7 + N)
    x = features(M, K, dt, M + K)
    w = torch.randn(N, K, generator=g) / math.sqrt(K)
    bias = torch.randn(N, generator=g) if N % 2 else None
    dy = torch.randn(M, N, generator=g).to(dt)
    xq, wq = to.mx4_round(x)[0].cuda(), to.mx4_round(w)[0].cuda()
    b64 = 0.0 if bias is None else bias.double().cuda()
    want = xq @ wq.t() + b64
    mass = xq.abs() @ wq.abs().t() + (0.0 if bias is None else b64.abs())
    w4 = quant.quantize_mx4(w.cuda())
    xc = x.cuda().requires_grad_()
    y = quant.mx4_linear(xc, w4, None if bias is None else bias.cuda())
    assert y.dtype == dt and y.shape == (M, N)
    assert bool(((y.double() - want).abs() <= bound(K, mass, want, dt)).all())
    dx, = torch.autograd.grad(y, xc, dy.cuda())
    d64 = dy.double().cuda()
    want, mass = d64 @ wq, d64.abs() @ wq.abs()
    assert dx.dtype == dt and dx.shape == (M, K)
    # an fp32 gradient is multiplied in three parts: three additions for each of the N terms
    assert bool(((dx.double() - want).abs() <= bound(3 * N, mass, want, dt)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
@pytest.mark.parametrize("M,K,N", [(1, 33000, 40), (3, 33100, 20), (100, 4096, 512), (700, 1100, 1300), (1, 300, 70000), (32, 8, 9),
                                   (7, 18432, 3000), (25, 9300, 3100), (1, 9300, 14400)])
def test_linear_long_sums_and_split_ones(hip_lib, dt, M, K, N):
    test_linear_forward_and_gradient(hip_lib, dt, M, K, N)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
def test_nan_scale_counts_whatever_the_codes(hip_lib, dt):
    from msf_wsi_amd import quant

    g = torch.Generator().manual_seed(4)
    q = quant.quantize_mx4(torch.randn(40, 600, generator=g).cuda())
    q.scales[1, 7, 2] = 255                                  # columns 320 ... 351 of row 7; the codes stay
    w = quant.MX4Tensor(q.codes, q.scales, 600)
    bad = torch.zeros(40, 600, dtype=torch.bool)
    bad[7, 320:352] = True
    assert torch.equal(w.dequantize(FP[dt]).isnan().cpu(), bad)
    for M in (1, 5, 40, 300):
        x = torch.randn(M, 600, generator=g).to(FP[dt]).cuda().requires_grad_()
        y = quant.mx4_linear(x, w)
        assert torch.equal(y.isnan().cpu(), bad.any(1).expand(M, 40))
        dx, = torch.autograd.grad(y, x, torch.randn(M, 40, generator=g).to(FP[dt]).cuda())
        assert torch.equal(dx.isnan().cpu(), bad.any(0).expand(M, 600))


@pytest.mark.gpu
def test_two_streams_at_once(hip_lib):
    """products that split their sums and share nothing but the weight, in flight on two streams together"""
    from msf_wsi_amd import quant

    w4 = quant.quantize_mx4(features(512, 4096, torch.float32, 8).cuda() / 30)
    xs = [features(M, 4096, torch.bfloat16, M).cuda().requires_grad_() for M in (100, 90)]
    dys = [features(x.shape[0], 512, torch.bfloat16, 3).cuda() for x in xs]

    def both(x, dy):
        y = quant.mx4_linear(x, w4)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    want = [both(x, dy) for x, dy in zip(xs, dys)]
    streams = [torch.cuda.Stream() for _ in xs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(both(xs[i], dys[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for pair in got[i] for a, b in zip(pair, want[i]))


@pytest.mark.gpu
@pytest.mark.parametrize("out", list(FP))
def test_linear_of_quantized_input_and_other_output_type(hip_lib, out):
    from msf_wsi_amd import quant

    x, w = features(40, 600, torch.bfloat16, 1).cuda(), features(70, 600, torch.float32, 2).cuda() / 25
    w4 = quant.quantize_mx4(w)
    a = quant.mx4_linear(x, w4, out_dtype=FP[out])
    b = quant.mx4_linear(quant.quantize_mx4(x), w4, out_dtype=FP[out])
    assert a.dtype == FP[out] and torch.equal(a, b)
    assert quant.mx4_linear(quant.quantize_mx4(x), w4).dtype == torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
@pytest.mark.parametrize("K,N", [(1, 1), (31, 5), (257, 33), (1001, 1537), (4608, 64)])
def test_one_row_is_a_row_of_many(hip_lib, dt, K, N):
    """a single row takes a path of its own: the same 4-bit values as the same row among others, NaN blocks included"""
    from msf_wsi_amd import quant

    x = features(3, K, FP[dt], K + N).cuda()
    w4 = quant.quantize_mx4(features(N, K, torch.float32, 5).cuda())
    many = quant.mx4_linear(x, w4, out_dtype=torch.float32)
    one = quant.mx4_linear(x[1:2], w4, out_dtype=torch.float32)
    mass = quant.quantize_mx4(x).dequantize().double().abs() @ w4.dequantize().double().abs().t()
    assert bool(((one.double() - many[1:2].double()).abs() <= 2 * (K + 8) * 2.0 ** -23 * mass[1:2]).all())
    assert torch.equal(quant.mx4_linear(x[1], w4, out_dtype=torch.float32), one[0])
    bad = x[1:2].clone()
    bad[0, K // 2] = math.inf
    assert quant.mx4_linear(bad, w4).isnan().all()


@pytest.mark.gpu
def test_weights_of_very_different_size(hip_lib):
    """scales up to 2^100 apart, in both operands' directions: every block's own scale counts"""
    from msf_wsi_amd import quant

    x = features(20, 512, torch.float32, 5)
    w = features(48, 512, torch.float32, 6)
    x[:, ::64] *= 2.0 ** -40
    w[::3] *= 2.0 ** 50
    w[1::3] *= 2.0 ** -50
    xq, wq = to.mx4_round(x)[0], to.mx4_round(w)[0]
    want, mass = xq @ wq.t(), xq.abs() @ wq.abs().t()
    xc = x.cuda().requires_grad_()
    y = quant.mx4_linear(xc, quant.quantize_mx4(w.cuda()))
    assert bool(((y.cpu().double() - want).abs() <= bound(512, mass, want, torch.float32)).all())
    for dt in FP.values():
        dy = features(20, 48, dt, 7).clamp(-100, 100)
        xc = x.to(torch.float32).cuda().requires_grad_()
        y = quant.mx4_linear(xc, quant.quantize_mx4(w.cuda()), out_dtype=dt)
        dx, = torch.autograd.grad(y, xc, dy.cuda())
        want, mass = dy.double() @ wq, dy.double().abs() @ wq.abs()
        assert bool(((dx.cpu().double() - want).abs() <= bound(3 * 48, mass, want, torch.float32)).all()), dt


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
def test_gradient_through_small_and_nan_weights(hip_lib, dt):
    """rows of W whose size alone decides an output (zeros of dy hide the others), over all scales; blocks of NaN"""
    from msf_wsi_amd import quant

    dt = FP[dt]
    e = torch.tensor([0, -20, -45, -70, -90, -8, 3, -60])
    w = torch.ldexp(features(8, 96, torch.float32, 20).clamp(-30, 30), e.view(8, 1))
    dy = torch.eye(8).to(dt) * 3
    w[6, 40] = math.inf
    w4 = quant.quantize_mx4(w.cuda())
    x = torch.zeros(8, 96, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(quant.mx4_linear(x, w4, out_dtype=dt), x, dy.cuda())
    want = 3 * to.mx4_round(w)[0]
    assert dx[:, 32:64].isnan().all()                      # 0 * NaN: the block of the weight reaches every row
    got = dx.cpu().double()
    got[:, 32:64], want[:, 32:64] = 0.0, 0.0
    assert torch.equal(got, want)                          # one term: exact


@pytest.mark.gpu
def test_gradient_by_differences(hip_lib):
    """the layer behind the rounding of x is linear: a step of x that stays on the 4-bit values moves y by exactly dx"""
    from msf_wsi_amd import quant

    levels = torch.tensor(to.LEVELS)
    g = torch.Generator().manual_seed(3)
    x = levels[torch.randint(0, 7, (6, 288), generator=g)].cuda()
    x[:, ::32] = 6.0                                        # fixes every block's scale at 1
    w4 = quant.quantize_mx4((torch.randn(10, 288, generator=g) / 16).cuda())
    c = torch.randn(6, 10, generator=g).cuda()
    xr = x.clone().requires_grad_()
    dx, = torch.autograd.grad((quant.mx4_linear(xr, w4) * c).sum(), xr)
    step = torch.zeros_like(x)
    step[:, 1] = torch.where(x[:, 1] < 2, 0.5, torch.where(x[:, 1] < 4, 1.0, 2.0))
    moved = ((quant.mx4_linear(x + step, w4).double() - quant.mx4_linear(x, w4).double()) * c.double()).sum()
    mass = (x.double().abs() + step.double()) @ w4.dequantize().double().abs().t()
    assert abs(float(moved) - float((dx * step).double().sum())) <= 4 * 300 * 2.0 ** -23 * float((mass * c.double().abs()).sum())


@pytest.mark.gpu
def test_layouts_streams_and_batches(hip_lib):
    from msf_wsi_amd import quant

    w4 = quant.quantize_mx4(features(96, 320, torch.float32, 8).cuda())
    x = features(30, 320, torch.bfloat16, 9).cuda()
    want = quant.mx4_linear(x, w4)
    assert torch.equal(quant.mx4_linear(x.view(5, 6, 320), w4).view(30, 96), want)
    wide = torch.zeros(30, 333, dtype=x.dtype, device="cuda")
    wide[:, 5:325] = x
    part = wide[:, 5:325].requires_grad_()
    y = quant.mx4_linear(part, w4)
    assert torch.equal(y, want)
    full, = torch.autograd.grad(y, part, torch.ones_like(y))
    xr = x.clone().requires_grad_()
    some, = torch.autograd.grad(quant.mx4_linear(xr, w4).sum(), xr)     # an expanded gradient: one value for all
    assert torch.equal(full, some)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = quant.mx4_linear(x, w4)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(1, 2304, 700), (40, 600, 300), (300, 1024, 520)])
def test_captured_forward_and_backward(hip_lib, M, K, N):
    from msf_wsi_amd import quant

    w4 = quant.quantize_mx4(features(N, K, torch.float32, 8).cuda() / 30)
    x = features(M, K, torch.bfloat16, 9).cuda().requires_grad_()
    dy = features(M, N, torch.bfloat16, 10).cuda()

    def both():
        y = quant.mx4_linear(x, w4)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        both()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = both()
    for seed in (11, 12, 13):
        with torch.no_grad():
            x.copy_(features(M, K, torch.bfloat16, seed))
            dy.copy_(features(M, N, torch.bfloat16, seed + 50))
        graph.replay()
        torch.cuda.synchronize()
        ey, edx = both()
        assert torch.equal(y, ey) and torch.equal(dx, edx)


@pytest.mark.gpu
def test_captured_split_sums(hip_lib):
    test_captured_forward_and_backward(hip_lib, 100, 4096, 512)


@pytest.mark.gpu
def test_refusals(hip_lib):
    from msf_wsi_amd import _lib, quant

    w4 = quant.quantize_mx4(torch.ones(8, 64, device="cuda"))
    with pytest.raises(ValueError):
        quant.mx4_linear(torch.zeros(2, 63, device="cuda"), w4)
    with pytest.raises(TypeError):
        quant.mx4_linear(torch.zeros(2, 64, device="cuda", dtype=torch.float64), w4)
    with pytest.raises(TypeError):
        quant.quantize_mx4(torch.zeros(2, 64, device="cuda", dtype=torch.int32))
    with pytest.raises(_lib.MsfwsiHipError):
        quant.mx4_linear(torch.zeros(2, 64), w4)
    with pytest.raises(ValueError):
        quant.mx4_linear(torch.zeros(2, 64, device="cuda"), w4, torch.zeros(8, device="cuda", requires_grad=True))
    with pytest.raises(TypeError):
        quant.mx4_linear(torch.zeros(2, 64, device="cuda"), w4, torch.zeros(8, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        quant.mx4_linear(torch.zeros(2, 64, device="cuda"), w4, torch.zeros(7, device="cuda"))
    with pytest.raises(ValueError):
        quant.MX4Tensor(w4.codes, w4.scales, 257)
    with pytest.raises(ValueError):
        quant.MX4Tensor(w4.codes, w4.scales[:, :4].contiguous(), 64)
    with pytest.raises(ValueError):
        quant.quantize_mx4(torch.zeros(3, 0, device="cuda"))
    x = torch.zeros(2, 64, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(quant.mx4_linear(x, w4).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.gpu
def test_offsets_past_31_bits(hip_lib):
    """70000 x 32000 bf16 (4.5 GB): quantised, widened and multiplied, the last rows as in a small tensor"""
    from msf_wsi_amd import quant

    x = torch.zeros(70000, 32000, dtype=torch.bfloat16, device="cuda")
    x[-3:] = features(3, 32000, torch.bfloat16, 1).cuda()
    q, few = quant.quantize_mx4(x), quant.quantize_mx4(x[-3:].clone())
    assert torch.equal(q.codes[:, -3:], few.codes) and torch.equal(q.scales[:, -3:], few.scales)
    assert torch.equal(q.dequantize(torch.bfloat16)[-3:], few.dequantize(torch.bfloat16))
    w4 = quant.quantize_mx4(features(40, 32000, torch.float32, 2).cuda() / 200)
    y, want = quant.mx4_linear(q, w4)[-3:].double(), quant.mx4_linear(few, w4).double()
    mass = few.dequantize().double().abs() @ w4.dequantize().double().abs().t()
    assert bool(((y - want).abs() <= 2 * 32008 * 2.0 ** -23 * mass).all())
    del x, q
    dy = torch.zeros(70000, 40, dtype=torch.bfloat16, device="cuda")
    dy[-3:] = 1.0
    w = quant.MX4Tensor(w4.codes, w4.scales, 32000)
    xr = torch.zeros(70000, 32000, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(quant.mx4_linear(xr, w), xr, dy)
    small, = torch.autograd.grad(quant.mx4_linear(xr[-3:], w), xr, torch.ones(3, 40, dtype=torch.bfloat16, device="cuda"))
    assert torch.equal(dx[-3:], small[-3:]) and float(dx[0].abs().max()) == 0.0


@pytest.mark.gpu
def test_changed_weights_are_noticed(hip_lib):
    """the gradient of a weight that was overwritten after the forward is refused, not computed from the new values"""
    from msf_wsi_amd import quant

    w4 = quant.quantize_mx4(torch.ones(8, 64, device="cuda"))
    x = torch.ones(2, 64, device="cuda", requires_grad=True)
    y = quant.mx4_linear(x, w4)
    w4.codes.zero_()
    with pytest.raises(RuntimeError):
        y.sum().backward()


@pytest.mark.gpu
def test_module_and_state(hip_lib):
    from msf_wsi_amd import quant

    torch.manual_seed(0)
    lin = torch.nn.Linear(200, 70).cuda()
    layer = quant.MX4Linear.from_linear(lin)
    x = torch.randn(9, 200, device="cuda")
    want = quant.mx4_linear(x, quant.quantize_mx4(lin.weight), lin.bias.detach())
    assert torch.equal(layer(x), want)
    other = quant.MX4Linear.from_linear(torch.nn.Linear(200, 70).cuda())
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), want) and not list(layer.parameters())


@pytest.mark.gpu
def test_module_cast_to_16_bits(hip_lib):
    from msf_wsi_amd import quant

    layer = quant.MX4Linear.from_linear(torch.nn.Linear(70, 30).cuda())
    x = features(5, 70, torch.bfloat16, 1).cuda()
    want = quant.mx4_linear(x, quant.MX4Tensor(layer.codes, layer.scales, 70), layer.bias.bfloat16().float())
    assert torch.equal(layer.bfloat16()(x), want)


def stored(scale_codes, seed):
    """a weight [rows, 64] of the given E, one a row, every code among its elements: (MX4Tensor, its values in float64)"""
    from msf_wsi_amd import quant

    rows = len(scale_codes)
    g = torch.Generator().manual_seed(seed)
    code = torch.randint(0, 16, (rows, 64), generator=g)
    code[:, :16] = torch.arange(16)
    codes = torch.zeros(1, rows, 128, dtype=torch.uint8)
    codes[0, :, :32] = (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8)
    e = torch.tensor(scale_codes)
    level = torch.tensor(to.LEVELS, dtype=torch.float64)
    values = torch.where(code > 7, -level[code % 8], level[code % 8]) * torch.exp2(e.double() - 127).view(rows, 1)
    scales = torch.zeros(1, rows, 8, dtype=torch.uint8)
    scales[0, :, :2] = e.view(rows, 1).to(torch.uint8)
    return quant.MX4Tensor(codes.cuda(), scales.cuda(), 64), values


def input_gradient(dy, w4):
    from msf_wsi_amd import kernels as kn

    dx = torch.empty(dy.shape[0], w4.shape[1], dtype=torch.float32, device="cuda")
    kn.mx4_dgrad(dy.cuda(), w4.codes, w4.scales, dx)
    return dx.cpu().double()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("E", [20, 40, 100, 107, 127, 150, 200, 252])
def test_gradient_over_the_whole_range_of_dy(hip_lib, dt, E):
    """every output is one product: exact but for the additions of an fp32 value's three parts (2^-23) and the smallest subnormal,
    and infinite only where the product itself is past the largest number"""
    dt = FP[dt]
    d = torch.tensor([3e38, -1e38, 1.7e37 * (1 + 2.0 ** -23), 1e30, 1.2345678, 2.0 ** -100 * (1 + 2.0 ** -23), 2.0 ** -115 * (1 + 2.0 ** -23),
                      -(2.0 ** -125) * 1.2345678, 2.0 ** -126 * (2 - 2.0 ** -23), 2.0 ** -130 * 1.2345678, 2.0 ** -140 * 1.2345678, 2.0 ** -149]).to(dt)
    w4, values = stored([E] * len(d), E)
    want = d.double().view(-1, 1) * values
    got = input_gradient(torch.diag(d), w4)
    fits = want.abs() <= torch.finfo(torch.float32).max * (1 - 2.0 ** -22)
    assert bool(((got - want).abs() <= 2.0 ** -23 * want.abs() + 2.0 ** -149)[fits].all())
    over = want.abs() > torch.finfo(torch.float32).max * (1 + 2.0 ** -22)
    assert bool(got[over].isinf().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
def test_gradient_of_scales_far_apart(hip_lib, dt):
    """all scales there are in the same columns; zeros of dy leave one weight to an output: exact, the smallest ones too"""
    w4, values = stored(list(range(253)), 1)
    assert torch.equal(input_gradient(torch.eye(253).to(FP[dt]), w4), values)
    some = [3, 0, 17, 110, 120]                              # close together, the smallest among them
    for k in range(1, 6):
        w4, values = stored(some[:k], k)
        assert torch.equal(input_gradient(torch.eye(k).to(FP[dt]) * 4, w4), values * 4)
    w4, values = stored([254, 253, 252, 2, 127], 2)
    d = torch.diag(torch.full((5,), 2.0 ** -10)).to(FP[dt])
    want = values * 2.0 ** -10
    assert bool(((input_gradient(d, w4) - want).abs() <= 2.0 ** -149).all())


@pytest.mark.gpu
def test_gradient_of_low_bits_beside_large_weights(hip_lib):
    """fp32: 24 bits from E = 16 up whatever stands beside them, 16 from E = 8, 8 below"""
    e = [0, 7, 8, 15, 16, 30, 252]
    w4, values = stored(e, 3)
    d = torch.full((7,), 1 + 2.0 ** -7 + 2.0 ** -15 + 2.0 ** -23)
    got, want = input_gradient(torch.diag(d), w4), values * float(d[0])
    for row, lost in enumerate([2.0 ** -7] * 2 + [2.0 ** -15] * 2 + [2.0 ** -23] * 3):
        assert bool(((got[row] - want[row]).abs() <= lost * want[row].abs() + 2.0 ** -149).all()), e[row]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(3, 33), (17, 300), (64, 1024)])
def test_widened_to_16_bits(hip_lib, rows, cols):
    """values rounded once to fp16 and bf16, large ones to infinity, small ones to subnormals and zero"""
    from msf_wsi_amd import quant

    x = features(rows, cols, torch.float32, rows) * torch.exp2(torch.linspace(-30, 20, rows)).view(-1, 1)
    q, v = quant.quantize_mx4(x.cuda()), to.mx4_round(x)[0]
    for dt in (torch.float16, torch.bfloat16):
        assert torch.equal(q.dequantize(dt).cpu(), v.to(dt))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 4, 20])
def test_products_of_all_scales(hip_lib, rows):
    """one product an output, scales from the smallest to the largest in both operands: exact, subnormal and infinite where the value is"""
    from msf_wsi_amd import kernels as kn

    e = [0, 1, 2, 40, 100, 126, 127, 128, 160, 230, 252, 253, 254]
    b4, b = stored(e, 5)
    for shift in range(0, len(e), 4):
        a4, a = stored((e[shift:] + e[:shift]) * rows, 6)
        only = torch.zeros(64, dtype=torch.bool)
        only[[5, 40]] = True                                # one element of either block, never both of an output
        keep = torch.zeros_like(a)
        odd = torch.arange(a.shape[0]) % 2
        keep[odd == 0, 5], keep[odd == 1, 40] = 1.0, 1.0
        codes = a4.codes.cpu()
        mask = torch.zeros(a.shape[0], 64, dtype=torch.uint8)
        mask[keep > 0] = 15
        codes[0, :, :32] &= mask[:, 0::2] | (mask[:, 1::2] << 4)
        y = torch.empty(a.shape[0], len(e), dtype=torch.float32, device="cuda")
        kn.mx4_gemm(codes.cuda(), a4.scales, b4.codes, b4.scales, 64, y)
        want = (a * keep) @ b.t()
        top = torch.finfo(torch.float32).max
        assert torch.equal(y.cpu().double().clamp(-2 * top, 2 * top), torch.where(want.abs() > top, torch.sign(want) * 2 * top, want.float().double()))


@pytest.mark.gpu
@pytest.mark.parametrize("arch,classes", [("resnet18", 1000), ("resnet50", 21)])
def test_resnet_with_a_4_bit_head(hip_lib, arch, classes):
    """the framework's own classifier as a frozen teacher: its head in 4 bits, its top logits, a student ResNet trained on them;
    and a 4-bit head on the student, which passes the gradient on to the encoder as the widened weight would"""
    from msf_wsi_amd import losses, quant
    from msf_wsi_amd.models import resnet

    torch.manual_seed(5)
    teacher, student = (getattr(resnet, arch)(num_classes=classes).cuda().train() for _ in range(2))
    x = torch.randn(4, 3, 64, 64, generator=torch.Generator().manual_seed(6)).cuda()
    fc, seen = teacher.fc, []
    teacher.fc = quant.MX4Linear.from_linear(fc)
    teacher.fc.register_forward_pre_hook(lambda module, args: seen.append(args[0]))
    with torch.no_grad():
        logits = teacher(x)
    feats, = seen
    w, b = teacher.fc, fc.bias.detach().double().cpu()
    wv = quant.MX4Tensor(w.codes, w.scales, w.in_features).dequantize().double().cpu()
    xq = to.mx4_round(feats.float().cpu())[0]
    want, mass = xq @ wv.t() + b, xq.abs() @ wv.abs().t() + b.abs()
    assert logits.shape == (4, classes) and bool(((logits.double().cpu() - want).abs() <= bound(w.in_features, mass, want, logits.dtype)).all())
    top = losses.top_logits(logits, 5, temperature=2.0)
    crit = losses.TopLogitDistillLoss(2.0)
    crit(student(x), top).backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in student.parameters())
    # the gradient of the features through a 4-bit head
    head = quant.MX4Linear.from_linear(student.fc)
    f = feats.detach().requires_grad_()
    y = head(f)
    dy, = torch.autograd.grad(crit(y, top), y, retain_graph=True)
    df, = torch.autograd.grad(y, f, dy)
    hv = quant.MX4Tensor(head.codes, head.scales, head.in_features).dequantize().double().cpu()
    want, mass = dy.double().cpu() @ hv, dy.double().cpu().abs() @ hv.abs()
    assert bool(((df.double().cpu() - want).abs() <= bound(3 * classes, mass, want, f.dtype)).all())
    student.zero_grad(set_to_none=True)
    student.fc = head
    crit(student(x), top).backward()
    assert not [n for n, _ in student.named_parameters() if n.startswith("fc.")]
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) and float(p.grad.abs().max()) > 0 for p in student.parameters())


@pytest.mark.gpu
@pytest.mark.parametrize("K,N", [(18432, 9216), (18000, 15000), (33000, 9000)])
def test_one_row_of_large_weights(hip_lib, K, N):
    """either side of the size up to which a single row takes one launch, against the widened weight in float64"""
    from msf_wsi_amd import quant

    w4 = quant.quantize_mx4(features(256, K, torch.float32, K).repeat((N + 255) // 256, 1)[:N].cuda() / 100)
    x = features(1, K, torch.bfloat16, N).cuda()
    y = quant.mx4_linear(x, w4, out_dtype=torch.float32)
    w, xq = w4.dequantize().double(), quant.quantize_mx4(x).dequantize().double()
    want, mass = xq @ w.t(), xq.abs() @ w.abs().t()
    assert bool(((y.double() - want).abs() <= bound(K, mass, want, torch.float32)).all())
