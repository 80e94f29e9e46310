"""Top logits and the distillation loss against float64.

Selection and order are exact.  Tolerances of the loss and its gradient, u = 2^-24 (half a step of fp32), A = the largest
|logit / T| distance of a row, n = classes:
  exponentials of arguments up to A are off by (A + 4) u relative (the argument's own rounding, then the function's), sums of n positive
  terms by at most n / 16 further roundings of a lane plus the tree, logarithms by 4 u absolute: every log q and log p is off by
  E = (3 A + n / 16 + 64) u absolute and every q, p by E relative.
  loss <= T^2 (sum p + p_r) E + rounding = T^2 E + u |loss|;   gradient <= |g| T E (q_j + p_j), then rounded once to its type."""
import math

import pytest
import torch

from oracle import teacher_oracle as to

FP = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24


def logits_of(rows, C, dt, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn(rows, C, generator=g)).to(dt)


def error_of(z, T):
    fin = torch.where(torch.isfinite(z.double()), z.double(), torch.zeros_like(z, dtype=torch.float64))
    return (3 * float((fin.amax(1) - fin.amin(1)).max()) / T + z.shape[1] / 16 + 64) * U


def check(z, values, indices, rest, mask, T, loss_rows, grad, dt, counts_scale=1.0):
    """kernel rows and gradients (of the sum of rows times counts_scale) against the definition"""
    want, wgrad, counts = to.distill(z.cpu(), values.cpu(), indices.cpu(), None if rest is None else rest.cpu(),
                                     None if mask is None else mask.cpu(), T)
    E = error_of(z.cpu(), T)
    if loss_rows is not None:
        got = loss_rows.cpu().double()
        bad = ~torch.isfinite(want)
        assert torch.equal(got[bad].isnan(), want[bad].isnan()) and torch.equal(got[bad & ~want.isnan()], want[bad & ~want.isnan()])
        assert bool(((got - want)[~bad].abs() <= T * T * E + 2 * U * want[~bad].abs()).all())
        assert bool((got[~counts] == 0).all())
    got = grad.cpu().double()
    nan = wgrad.isnan()
    assert torch.equal(got.isnan(), nan)
    assert bool((got[~counts] == 0).all())
    # sum of the shares and of q bounds the size of what is subtracted
    q = torch.softmax(z.cpu().double() / T, 1).nan_to_num(0.0)
    p = torch.zeros(q.shape[0], q.shape[1] + 1, dtype=torch.float64)
    idx = indices.cpu().long().clamp(min=-1)
    logs = torch.where(idx >= 0, values.cpu().double() / T, torch.full(values.shape, -math.inf, dtype=torch.float64))
    if rest is not None:
        logs = torch.cat([logs, rest.cpu().double().view(-1, 1)], 1)
    share = torch.softmax(logs, 1).nan_to_num(0.0)
    p.scatter_add_(1, torch.where((idx >= 0) & (idx < q.shape[1]), idx, q.shape[1]), share[:, :idx.shape[1]])
    p = p[:, :-1]
    spread = share[:, idx.shape[1]:].sum(1, keepdim=True) * torch.softmax(torch.where(p > 0, -math.inf, z.cpu().double() / T), 1).nan_to_num(0.0)
    size = T * counts_scale * (q + p + spread)
    tiny = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[dt]
    lim = size * E * 2 + torch.finfo(dt).eps / 2 * (wgrad * counts_scale).abs() * (1 + 1e-5) + tiny
    err = (got - wgrad * counts_scale)[~nan].abs()
    assert bool((err <= lim[~nan]).all()), float((err / lim[~nan]).max())


# ---- CPU -------------------------------------------------------------------------------------------------------------
def test_oracle_by_hand_and_by_differences():
    v, i, r = to.top_logits(torch.tensor([[1.0, 3.0, 3.0, math.nan, -math.inf]]), 3, 1.0)
    assert i.tolist() == [[3, 1, 2]] and v[0, 1:].tolist() == [3.0, 3.0] and abs(float(r) - 1.0) < 1e-15
    # two classes listed in full: the loss is the divergence itself
    z, t = torch.tensor([[0.3, -0.2]]), torch.tensor([[2.0, 1.0]])
    loss, grad, counts = to.distill(z, t, torch.tensor([[0, 1]]), None, None, 1.0)
    p, q = torch.softmax(t.double(), 1), torch.softmax(z.double(), 1)
    assert abs(float(loss) - float((p * (p / q).log()).sum())) < 1e-15 and torch.allclose(grad, q - p) and bool(counts.all())
    z = logits_of(4, 9, torch.float32, 1).double()
    values, indices, rest = to.top_logits(logits_of(4, 9, torch.float32, 2), 3, 2.0)
    indices[1, 2], indices[2] = indices[1, 0], -1
    _, grad, _ = to.distill(z, values, indices, rest, None, 2.0)
    for c in range(9):
        h = torch.zeros_like(z)
        h[:, c] = 1e-5
        up, dn = (to.distill(z + s * h, values, indices, rest, None, 2.0)[0] for s in (1, -1))
        assert torch.allclose((up - dn) / 2e-5, grad[:, c], atol=1e-8)


def test_refusals_without_a_gpu(hip_lib):
    from msf_wsi_amd import _lib, losses

    with pytest.raises(_lib.MsfwsiHipError):
        losses.top_logits(torch.zeros(2, 5), 2)
    with pytest.raises(_lib.MsfwsiHipError):
        losses.TopLogitDistillLoss()(torch.zeros(2, 5), losses.TopLogits(torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int32)))
    for t in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            losses.TopLogitDistillLoss(temperature=t)
    with pytest.raises(ValueError):
        losses.TopLogitDistillLoss(reduction="batchmean")
    assert hip_lib.msfwsi_top_logits(0, None, 5, 1, 5, 1, 6, 1.0, None, None, None, None, None) == -1       # k > classes
    assert hip_lib.msfwsi_top_logits(0, None, 5, 1, 5, 1, 2, 1.0, None, None, None, None, None) == -1       # no memory
    assert hip_lib.msfwsi_top_logits(0, None, 4, 2, 5, 1, 2, 1.0, None, None, None, None, None) == -1       # rows overlap
    assert hip_lib.msfwsi_top_logits(0, None, 5, 0, 5, 1, 2, 1.0, None, None, None, None, None) == 0        # no rows
    assert hip_lib.msfwsi_distill_fwd(0, None, 5, 1, 5, 1, 65, None, None, None, None, 1.0, 1, None, None, None, None, None, None) == -1
    assert hip_lib.msfwsi_distill_bwd(3, None, 5, 1, 5, 1, 2, None, None, None, 1.0, None, None, None, 0, None, None) == -1


# ---- GPU: selection --------------------------------------------------------------------------------------------------
ROWS = [(1, 1, 1), (3, 2, 2), (5, 33, 7), (70, 64, 3), (4, 65, 64), (9, 257, 33), (33, 1000, 10), (2, 1001, 64), (3, 8191, 32), (2, 65536, 16),
        (1, 65539, 64), (2, 131072, 5)]


def same_top(x, k, T, got):
    v, i, r = to.top_logits(x, k, T)
    assert torch.equal(got.indices.cpu().long(), i)
    assert torch.equal(got.values.cpu().double().nan_to_num(nan=9e9), v.nan_to_num(nan=9e9))
    rest = got.rest.cpu().double()
    fin = torch.isfinite(r)
    assert torch.equal(rest[~fin].nan_to_num(nan=9e9), r[~fin].nan_to_num(nan=9e9))
    E = error_of(x, T)
    assert bool(((rest - r)[fin].abs() <= E + 2 * U * r[fin].abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
@pytest.mark.parametrize("rows,C,k", ROWS)
def test_top_logits_rows(hip_lib, dt, rows, C, k):
    from msf_wsi_amd import losses

    x = logits_of(rows, C, FP[dt], rows + C + k)
    same_top(x, k, 0.5, losses.top_logits(x.cuda(), k, temperature=0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("C", [40, 1000, 20011])
@pytest.mark.parametrize("kind", ["ascending", "descending", "equal", "few", "masked", "nan", "zeros", "one block"])
def test_top_logits_orders(hip_lib, kind, C):
    """orders and ties that a selection by thresholds or by halves could trip over"""
    from msf_wsi_amd import losses

    g = torch.Generator().manual_seed(C)
    k = 33
    if kind == "ascending":
        x = torch.arange(C).float().repeat(2, 1) / 64 - 5
    elif kind == "descending":
        x = -torch.arange(C).float().repeat(2, 1) / 64
    elif kind == "equal":
        x = torch.full((2, C), -1.5)
    elif kind == "few":                      # three values: long ties across the border
        x = torch.randint(0, 3, (2, C), generator=g).float()
    elif kind == "masked":                   # fewer finite logits than k; a row with none
        x = torch.full((2, C), -math.inf)
        x[0, C // 2:C // 2 + 5] = torch.randn(5, generator=g)
    elif kind == "nan":
        x = torch.randn(3, C, generator=g)
        x[0, 7], x[1, C - 1], x[1, 3], x[2, 11], x[2, 12] = math.nan, -math.nan, math.inf, math.inf, -math.inf
        x[1, 5:39] = math.nan                # more of them than k: rest is NaN
    elif kind == "zeros":                    # -0 and +0 are equal
        x = torch.where(torch.rand(2, C, generator=g) < 0.5, -0.0, 0.0)
    else:                                    # every large value next to the others
        x = torch.randn(2, C, generator=g)
        x[:, 2:38] += 50.0
    same_top(x, k, 1.0, losses.top_logits(x.cuda(), k))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
@pytest.mark.parametrize("shape,k", [((2, 6, 9, 7), 6), ((3, 21, 16, 16), 4), ((1, 64, 5), 16), ((2, 40, 300), 20), ((4, 3, 1, 1), 2)])
def test_top_logits_maps(hip_lib, dt, shape, k):
    from msf_wsi_amd import losses

    x = logits_of(shape[0] * math.prod(shape[2:]), shape[1], FP[dt], sum(shape)).view(shape[0], *shape[2:], shape[1]).movedim(-1, 1)
    last = x.movedim(1, -1).reshape(-1, shape[1])
    for form in [x.contiguous().cuda(), x.cuda()] + ([x.contiguous(memory_format=torch.channels_last).cuda()] if x.dim() == 4 else []):
        got = losses.top_logits(form, k, temperature=2.0, dim=1)
        assert got.values.shape == (shape[0], k) + shape[2:] and got.rest.shape == (shape[0],) + shape[2:]
        flat = losses.TopLogits(got.values.movedim(1, -1).reshape(-1, k), got.indices.movedim(1, -1).reshape(-1, k), got.rest.reshape(-1))
        same_top(last, k, 2.0, flat)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,C", [("fp32", 300001), ("bf16", 540003)])
def test_top_logits_many_segments(hip_lib, dt, C):
    """more list entries than a merge holds at once"""
    test_top_logits_rows(hip_lib, dt, 2, C, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
def test_maps_of_many_classes(hip_lib, dt):
    """maps whose class index takes more than 16 bits, lists of every length class"""
    for k in (3, 9, 40):
        test_top_logits_maps(hip_lib, dt, (1, 70001, 3), k)
        test_loss_maps(hip_lib, dt, (1, 70001, 3), k)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
@pytest.mark.parametrize("rows,C,k", [(300, 1, 1), (4100, 16, 4), (9000, 33, 7), (16500, 16, 16), (33000, 128, 3), (5000, 300, 40), (70, 2000, 64)])
def test_many_short_rows(hip_lib, dt, rows, C, k):
    """rows that a thread takes each, and long lists from rows that a wave takes; some of the rows are checked"""
    from msf_wsi_amd import losses

    T = 2.0
    z, t = logits_of(rows, C, FP[dt], rows + C), logits_of(rows, C, FP[dt], rows * C + k)
    teacher = losses.top_logits(t.cuda(), k, T)
    pick = sorted({0, 1, 63, 64, 255, 256, rows // 2, rows - 2, rows - 1} & set(range(rows)))
    some = losses.TopLogits(*(a[pick] for a in teacher))
    same_top(t[pick], k, T, some)
    zc = z.cuda().requires_grad_()
    row = losses.TopLogitDistillLoss(T, "none")(zc, teacher)
    grad, = torch.autograd.grad(row, zc, torch.ones(rows, device="cuda"))
    check(z[pick], some.values, some.indices, some.rest, None, T, row.detach()[pick], grad[pick], FP[dt])
    mean = losses.TopLogitDistillLoss(T)(zc, teacher)
    want = float(row.detach().double().mean())
    assert abs(mean.item() - want) <= 4 * U * abs(want) + 1e-30


@pytest.mark.gpu
@pytest.mark.parametrize("C", [40, 129])
def test_more_rows_than_2_to_the_24(hip_lib, C):
    from msf_wsi_amd import losses

    z = torch.zeros(2 ** 24 + 77, C, dtype=torch.bfloat16, device="cuda")
    pick = [0, 2 ** 24 - 2, 2 ** 24 - 1, 2 ** 24, 2 ** 24 + 76]
    small = logits_of(5, C, torch.bfloat16, 3)
    z[pick] = small.cuda()
    teacher = losses.top_logits(z, 2)
    some = losses.TopLogits(*(a[pick] for a in teacher))
    same_top(small, 2, 1.0, some)
    z[pick] = z[pick].flip(1)
    z.requires_grad_()
    row = losses.TopLogitDistillLoss(reduction="none")(z, teacher)
    grad, = torch.autograd.grad(row, z, torch.ones_like(row))
    check(small.flip(1), some.values, some.indices, some.rest, None, 1.0, row.detach()[pick], grad[pick], torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
def test_top_logits_repeat_bit_for_bit(hip_lib, dt):
    """also where many candidates compete for places (coarse values: ties everywhere)"""
    from msf_wsi_amd import losses

    x = torch.cat([logits_of(40, 30011, FP[dt], 5), (logits_of(40, 30011, torch.float32, 6) * 4).round().to(FP[dt])]).cuda()
    first = losses.top_logits(x, 48, 2.0)
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(first, losses.top_logits(x, 48, 2.0)))


@pytest.mark.gpu
def test_masks_of_the_lowest_value(hip_lib):
    """logits masked with the type's lowest number instead of -inf: as -inf beside others, uniform where nothing else is left"""
    from msf_wsi_amd import losses

    for dt in FP.values():
        low = torch.finfo(dt).min
        z = torch.full((3, 900), low, dtype=dt)
        z[0, 3:9], z[1] = 0.5, -math.inf
        z[1, 7] = 1.0
        top = losses.top_logits(z.cuda(), 4, 2.0)
        assert top.indices.tolist() == [[3, 4, 5, 6], [7, 0, 1, 2], [0, 1, 2, 3]]
        assert abs(float(top.rest[0]) - (0.25 + math.log(2))) < 1e-6 and float(top.rest[1]) == -math.inf
        teacher = losses.TopLogits(torch.zeros(3, 2, device="cuda"), torch.tensor([[3, 4]] * 3, dtype=torch.int32, device="cuda"))
        zc = z[[0, 2]].cuda().requires_grad_()
        crit = losses.TopLogitDistillLoss(2.0, "none")
        row = crit(zc, losses.TopLogits(*(t[:2] for t in teacher[:2])))
        want = [4.0 * math.log(6 / 2), 4.0 * math.log(900 / 2)]      # T^2 (log 1/2 - log q) with q = 1/6, 1/900
        assert all(abs(a - b) < 1e-4 for a, b in zip(row.tolist(), want))
        g, = torch.autograd.grad(row, zc, torch.ones(2, device="cuda"))
        # A probability is a product of two powers of 2 whose exponents hold log2(s), s up to 900: at most 1.5 steps of 2^-20 off (one
        # of the logarithm, half of its rounding), so 1.5 ln 2 2^-20; the two powers, a step of 2^-23 each, and four roundings of
        # 2^-24 follow.  Together under 13 2^-23 of the value.  The teacher's 1/2 has log2(2) in its exponent: under 4 2^-23.
        half, f32 = torch.finfo(dt).eps / 2, 2.0 ** -23
        assert abs(float(g[1, 10]) - 2.0 / 900) <= (half + 13 * f32) * 2.0 / 900
        assert abs(float(g[1, 3]) - 2.0 * (1 / 900 - 0.5)) <= half + 4 * f32
        assert float(g[0, 10]) == 0.0 and abs(float(g[0, 8]) - 2.0 / 6) <= (half + 13 * f32) / 3


@pytest.mark.gpu
def test_offsets_past_31_bits(hip_lib):
    """33000 x 65600 bf16 logits (4.3 GB): the last rows, and the rows either side of 2^31 elements, as in a small tensor"""
    from msf_wsi_amd import losses

    rows, C = 33000, 65600
    z = torch.zeros(rows, C, dtype=torch.bfloat16, device="cuda")
    pick = [0, 32734, 32735, 32736, rows - 1]
    z[pick] = logits_of(5, C, torch.bfloat16, 77).cuda()
    small = z[pick].clone()
    big, few = losses.top_logits(z, 6, 2.0), losses.top_logits(small, 6, 2.0)
    assert all(torch.equal(a[pick], b) for a, b in zip(big, few))
    del big
    teacher = losses.TopLogits(few.values.new_zeros(rows, 6), few.indices.new_zeros(rows, 6), None)
    teacher.values[pick], teacher.indices[pick] = few.values, few.indices
    mask = torch.zeros(rows, dtype=torch.bool, device="cuda")
    mask[pick] = True
    crit = losses.TopLogitDistillLoss(2.0, "sum")
    zr, sr = z.requires_grad_(), small.requires_grad_()
    a, b = crit(zr, teacher, mask), crit(sr, losses.TopLogits(few.values, few.indices))
    assert abs(a.item() - b.item()) <= 4 * U * abs(b.item())
    ga, gb = torch.autograd.grad(a, zr)[0], torch.autograd.grad(b, sr)[0]
    assert torch.equal(ga[pick], gb) and float(ga[1].abs().max()) == 0.0


@pytest.mark.gpu
def test_top_logits_slices_and_refusals(hip_lib):
    from msf_wsi_amd import losses

    wide = logits_of(6, 1050, torch.bfloat16, 3)
    part = wide.cuda()[:, 3:1034]
    same_top(wide[:, 3:1034], 20, 1.0, losses.top_logits(part, 20))
    assert losses.top_logits(torch.zeros(0, 7, device="cuda"), 3).values.shape == (0, 3)
    assert losses.top_logits(torch.zeros(2, 7, 0, device="cuda"), 3, dim=1).indices.shape == (2, 3, 0)
    one = losses.top_logits(torch.tensor([1.0, 5.0, 2.0], device="cuda"), 2)
    assert one.indices.tolist() == [1, 2] and one.rest.shape == ()
    x = torch.zeros(2, 70, device="cuda")
    for bad in (0, 65, 71):
        with pytest.raises(ValueError):
            losses.top_logits(x, bad)
    with pytest.raises(ValueError):
        losses.top_logits(torch.zeros(2, 3, 4, 5, device="cuda"), 1, dim=2)
    with pytest.raises(TypeError):
        losses.top_logits(x.double(), 3)
    with pytest.raises(ValueError):
        losses.top_logits(x, 3, temperature=0.0)


# ---- GPU: the loss ---------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
@pytest.mark.parametrize("with_rest", [False, True])
@pytest.mark.parametrize("rows,C,k", ROWS)
def test_loss_rows(hip_lib, dt, with_rest, rows, C, k):
    from msf_wsi_amd import losses

    T = 2.0
    z, t = logits_of(rows, C, FP[dt], rows + C), logits_of(rows, C, torch.float32, rows * C + k)
    v, i, r = to.top_logits(t, k, T)
    teacher = losses.TopLogits(v.float().cuda(), i.int().cuda(), r.float().cuda() if with_rest else None)
    g = torch.Generator().manual_seed(k)
    mask = torch.rand(rows, generator=g) < 0.7 if rows > 3 else None
    cm = None if mask is None else mask.cuda()
    zc = z.cuda().requires_grad_()
    rows_loss = losses.TopLogitDistillLoss(T, "none")(zc, teacher, cm)
    grad, = torch.autograd.grad(rows_loss, zc, torch.ones(rows, device="cuda"))
    check(z, teacher.values, teacher.indices, teacher.rest, mask, T, rows_loss.detach(), grad, FP[dt])
    total = losses.TopLogitDistillLoss(T, "sum")(zc, teacher, cm)
    mean = losses.TopLogitDistillLoss(T)(zc, teacher, cm)
    n = rows if mask is None else int(mask.sum())
    want = float(rows_loss.detach().double().sum())
    assert abs(float(total) - want) <= 2 * U * abs(want) + 1e-30 and abs(float(mean) - want / max(n, 1)) <= 4 * U * abs(want) + 1e-30
    sgrad, = torch.autograd.grad(total, zc, torch.tensor(256.0, device="cuda"))
    check(z, teacher.values, teacher.indices, teacher.rest, mask, T, None, sgrad, FP[dt], 256.0)
    mgrad, = torch.autograd.grad(mean, zc, torch.tensor(256.0, device="cuda"))
    check(z, teacher.values, teacher.indices, teacher.rest, mask, T, None, mgrad, FP[dt], 256.0 / max(n, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
@pytest.mark.parametrize("shape,k", [((2, 6, 9, 7), 6), ((3, 21, 16, 16), 4), ((1, 64, 5), 16), ((2, 40, 300), 20)])
def test_loss_maps(hip_lib, dt, shape, k):
    from msf_wsi_amd import losses

    T, n = 1.0, shape[0] * math.prod(shape[2:])
    z, t = logits_of(n, shape[1], FP[dt], 5), logits_of(n, shape[1], torch.float32, 6)
    v, i, r = to.top_logits(t, k, T)
    mask = torch.rand(n, generator=torch.Generator().manual_seed(1)) < 0.5

    def to_map(a, last):
        return a.view(shape[0], *shape[2:], last).movedim(-1, 1)

    where = (shape[0],) + shape[2:]
    teacher = losses.TopLogits(to_map(v.float(), k).cuda(), to_map(i.int(), k).contiguous().cuda(), r.float().view(where).cuda())
    zm = to_map(z, shape[1])
    for form in [zm.contiguous(), zm] + ([zm.contiguous(memory_format=torch.channels_last)] if zm.dim() == 4 else []):
        zc = form.cuda().requires_grad_()
        row = losses.TopLogitDistillLoss(T, "none", dim=1)(zc, teacher, mask.view(where).cuda())
        assert row.shape == where
        grad, = torch.autograd.grad(row.sum(), zc)
        check(z, v.float(), i, r.float(), mask, T, row.detach().reshape(-1), grad.movedim(1, -1).reshape(n, -1), FP[dt])


def special_case():
    """one row for every way the inputs can be odd; (z, values, indices, rest, mask)"""
    C, k = 300, 4
    z, t = logits_of(16, C, torch.float32, 11), logits_of(16, C, torch.float32, 12)
    v, i, r = to.top_logits(t, k, 1.0)
    v, i, r = v.float(), i.int(), r.float()
    mask = torch.ones(16, dtype=torch.bool)
    i[1] = -1                                               # padding only, but a rest: everything is the rest
    i[2], r[2] = -1, -math.inf                              # nothing at all
    v[3], r[3] = -math.inf, -math.inf                       # listed classes without mass, no rest
    i[4, 2:] = -1                                           # a shorter list
    i[5, 1] = i[5, 0]                                       # the same class twice
    z[6, 50:] = -math.inf                                   # masked student classes, listed ones among them
    i[6] = torch.tensor([3, 7, 200, 9], dtype=torch.int32)
    z[7] = -math.inf                                        # a student row that is masked out whole
    z[8, 17], mask[8] = math.nan, False                     # NaN where nothing counts
    v[8], i[8], r[8] = math.nan, 10 ** 9, math.nan
    i[9, 3] = C                                             # past the classes
    z[10, 5] = math.nan                                     # NaN that counts
    v[11, 2] = -math.inf                                    # a listed class without mass
    z[12] = z[12].abs().neg() - 1e4                         # far from zero
    z[13, int(i[13, 0])] = 80.0                             # sure of the first class: almost nothing left for the others
    z[14] = torch.finfo(torch.float32).min                  # a mask of the type's lowest value
    z[14, 3:9] = 0.5
    i[14], v[14] = torch.tensor([3, 4, 5, 6], dtype=torch.int32), 0.0
    return z, v, i, r, mask


@pytest.mark.gpu
def test_loss_odd_rows(hip_lib):
    from msf_wsi_amd import losses

    z, v, i, r, mask = special_case()
    for layout in ("rows", "maps"):
        zl, vl, il = (a.t()[None].contiguous() if layout == "maps" else a for a in (z, v, i))
        shape = (1, 16) if layout == "maps" else (16,)
        zc = zl.cuda().requires_grad_()
        crit = losses.TopLogitDistillLoss(1.0, "none", dim=1 if layout == "maps" else -1)
        row = crit(zc, losses.TopLogits(vl.cuda(), il.cuda(), r.view(shape).cuda()), mask.view(shape).cuda())
        grad, = torch.autograd.grad(row, zc, torch.ones_like(row))
        row, grad = row.detach().reshape(-1), (grad[0].t() if layout == "maps" else grad)
        want, wgrad, counts = to.distill(z, v, i, r, mask, 1.0)
        assert counts.tolist() == [True, True] + [False] * 2 + [True] * 4 + [False] + [True] * 7
        assert row.isnan().tolist() == [j in (9, 10) for j in range(16)]
        assert torch.isinf(row).tolist() == [j in (6, 7) for j in range(16)]
        fin = [0, 1, 4, 5, 11, 12, 13, 14, 15]
        for j in (2, 3, 8):
            assert float(row[j]) == 0.0 and float(grad[j].abs().max()) == 0.0
        zz = torch.where(torch.isfinite(z[fin]), z[fin], torch.zeros(()))
        near = zz.clone()
        near[fin.index(14)] = near[fin.index(14)].clamp(min=-100)      # the size of the error there is that of the finite part
        E = error_of(near, 1.0)
        assert bool(((row[fin].cpu().double() - want[fin]).abs() <= E + 2 * U * want[fin].abs()).all())
        assert bool(((grad[fin].cpu().double() - wgrad[fin]).abs() <= 4 * E).all())
        # the row with masked classes: finite gradients, zero outside list and mask
        assert bool(torch.isfinite(grad[6]).all()) and float(grad[6, 250]) == 0.0
        assert bool(((grad[6].cpu().double() - wgrad[6]).abs() <= 4 * E).all()) and bool(((grad[7].cpu().double() - wgrad[7]).abs() <= 4 * E).all())
        assert grad[9].isnan().all() and grad[10].isnan().all()
        crit = losses.TopLogitDistillLoss(1.0, "mean", dim=1 if layout == "maps" else -1)
        keep = mask.clone()
        keep[[6, 7, 9, 10]] = False
        m = crit(zc, losses.TopLogits(vl.cuda(), il.cuda(), r.view(shape).cuda()), keep.view(shape).cuda())
        assert abs(float(m) - float(row[fin].double().mean())) <= 4 * U * float(row[fin].double().mean())
        none = crit(zc, losses.TopLogits(vl.cuda(), il.cuda(), r.view(shape).cuda()), torch.zeros(shape, dtype=torch.bool, device="cuda"))
        gone, = torch.autograd.grad(none, zc)
        assert float(none) == 0.0 and float(gone.abs().max()) == 0.0


@pytest.mark.gpu
def test_loss_per_row_gradients_slices_and_repeats(hip_lib):
    from msf_wsi_amd import losses

    z, t = logits_of(12, 517, torch.bfloat16, 21), logits_of(12, 517, torch.float32, 22)
    v, i, r = to.top_logits(t, 5, 0.5)
    v, i, r = v.float().cuda(), i.int().cuda(), r.float().cuda()
    w = torch.randn(12, generator=torch.Generator().manual_seed(2)).cuda()
    crit = losses.TopLogitDistillLoss(0.5, "none")
    wide = torch.zeros(12, 531, dtype=torch.bfloat16, device="cuda")
    wide[:, 7:524] = z.cuda()
    part = wide[:, 7:524].requires_grad_()
    zc = z.cuda().requires_grad_()
    a, b = crit(zc, losses.TopLogits(v, i, r)), crit(part, losses.TopLogits(v, i, r))
    ga, gb = torch.autograd.grad(a, zc, w)[0], torch.autograd.grad(b, part, w)[0]
    assert torch.equal(a, b) and torch.equal(ga, gb)
    for again in range(3):                                   # the same call gives the same bits
        assert torch.equal(crit(zc, losses.TopLogits(v, i, r)), a)
    one = torch.autograd.grad(crit(zc, losses.TopLogits(v, i, r)), zc, torch.ones(12, device="cuda"))[0]
    assert bool(((ga.double() - one.double() * w.double()[:, None]).abs() <= 2.0 ** -7 * (one.double() * w.double()[:, None]).abs() + 1e-30).all())
    zs = z.cuda()[3:9].detach().requires_grad_()             # slices of a batch, at any alignment
    part = crit(zs, losses.TopLogits(v[3:9], i[3:9], r[3:9]), torch.ones(12, dtype=torch.bool, device="cuda")[5:11])
    assert torch.equal(part, a[3:9])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = crit(zc, losses.TopLogits(v, i, r))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, a)


@pytest.mark.gpu
def test_loss_empty_and_refused(hip_lib):
    from msf_wsi_amd import losses

    f32, i32 = dict(device="cuda"), dict(device="cuda", dtype=torch.int32)
    z = torch.zeros(0, 9, requires_grad=True, **f32)
    loss = losses.TopLogitDistillLoss()(z, losses.TopLogits(torch.zeros(0, 2, **f32), torch.zeros(0, 2, **i32)))
    loss.backward()
    assert float(loss) == 0.0 and z.grad.shape == (0, 9)
    z = torch.zeros(3, 9, requires_grad=True, **f32)
    v, i = torch.zeros(3, 2, **f32), torch.zeros(3, 2, **i32)
    crit, TL = losses.TopLogitDistillLoss(), losses.TopLogits
    for bad in (TL(v[:2], i[:2]), TL(v, i[:, :1]), TL(v, i, torch.zeros(2, **f32)), TL(v, i, torch.zeros(3, device="cuda", dtype=torch.float64)),
                TL(torch.zeros(3, 65, **f32), torch.zeros(3, 65, **i32)), TL(torch.zeros(3, 0, **f32), torch.zeros(3, 0, **i32)),
                TL(v.clone().requires_grad_(), i)):
        with pytest.raises(ValueError):
            crit(z, bad)
    for bad in (TL(v, i.long()), TL(v.half(), i)):
        with pytest.raises(TypeError):
            crit(z, bad)
    with pytest.raises(ValueError):
        crit(z, TL(v, i), torch.ones(3, device="cuda"))
    with pytest.raises(TypeError):
        crit(z.double(), TL(v, i))
    with pytest.raises(ValueError):
        losses.TopLogitDistillLoss(dim=2)(torch.zeros(2, 3, 4, 5, **f32), TL(v, i))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dim", [((40, 1000), -1), ((2, 21, 24, 24), 1), ((3, 70001), -1)])
def test_captured_selection_and_loss(hip_lib, shape, dim):
    from msf_wsi_amd import losses

    C = shape[dim]
    t = logits_of(math.prod(shape) // C, C, torch.bfloat16, 30).cuda().view(shape)
    z = logits_of(math.prod(shape) // C, C, torch.bfloat16, 31).cuda().view(shape).requires_grad_()
    crit = losses.TopLogitDistillLoss(2.0, dim=dim)

    def step():
        top = losses.top_logits(t, 8, 2.0, dim=dim)
        loss = crit(z, top)
        return tuple(top) + (loss.detach(), torch.autograd.grad(loss, z)[0])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (32, 33, 34):
        with torch.no_grad():
            t.copy_(logits_of(math.prod(shape) // C, C, torch.bfloat16, seed).view(shape))
            z.copy_(logits_of(math.prod(shape) // C, C, torch.bfloat16, seed + 9).view(shape))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.gpu
def test_frozen_teacher_chain(hip_lib):
    """as they are used together: a 4-bit teacher head, its top logits, the loss of a student that ends in a 4-bit head of its
    own, and the gradient of the student's features against float64 through the same 4-bit values"""
    from msf_wsi_amd import losses, quant

    torch.manual_seed(3)
    head = torch.nn.Linear(512, 1500).cuda()
    teacher, student = quant.MX4Linear.from_linear(head), quant.MX4Linear.from_linear(torch.nn.Linear(512, 1500).cuda())
    feats = torch.randn(24, 512, device="cuda")
    with torch.no_grad():
        top = losses.top_logits(teacher(feats), 12, temperature=2.0)
    x = torch.randn(24, 512, device="cuda", requires_grad=True)
    logits = student(x)
    loss = losses.TopLogitDistillLoss(2.0)(logits, top)
    loss.backward()
    w = quant.MX4Tensor(student.codes, student.scales, 512).dequantize().cpu().double()
    y = to.mx4_round(x.detach().cpu())[0] @ w.t() + student.bias.cpu().double()
    rows, grad, _ = to.distill(y, top.values.cpu(), top.indices.cpu(), top.rest.cpu(), None, 2.0)
    # the logits' own error (520 * 2^-23 of their mass) moves log q by twice as much, the gradient by as much of q
    mass = to.mx4_round(x.detach().cpu())[0].abs() @ w.abs().t() + student.bias.cpu().double().abs()
    dy = 520 * 2.0 ** -23 * float(mass.max())
    assert abs(float(loss) - float(rows.mean())) <= 4.0 * (2 * dy / 2.0 + error_of(y, 2.0))
    want = grad @ w / 24
    lim = (2 * dy + 2 * error_of(y, 2.0)) * 2.0 * 3 * float(w.abs().max()) / 24 + 1508 * 3 * 2.0 ** -23 * float((grad.abs() @ w.abs()).max()) / 24
    assert float((x.grad.cpu().double() - want).abs().max()) <= lim


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
@pytest.mark.parametrize("rows,C,k", [(10300, 40, 2), (6, 40, 2), (6, 900, 33), (6, 2000, 5), (6, 20011, 3), (6, 300001, 64)])
def test_infinite_logits_left_over(hip_lib, dt, rows, C, k):
    """+inf outside the list makes rest +inf, one or several of them, together or apart; a NaN outside makes it NaN"""
    from msf_wsi_amd import losses

    g = torch.Generator().manual_seed(C)
    x = logits_of(rows, C, FP[dt], C)
    at = [torch.randperm(C, generator=g) for _ in range(6)]
    x[0, at[0][:k + 1]] = math.inf                          # one left over
    x[1, at[1][:k + 3]] = math.inf
    x[2, 1:k + 3] = math.inf                                # next to each other
    x[3, at[3][:k + 1]], x[3, at[3][k + 1]] = math.inf, math.nan                 # the NaN is listed
    x[4, at[4][:k + 2]], x[4, at[4][k + 2:k + 5]] = math.nan, math.inf           # NaN and +inf left over
    x[5, at[5][:k]] = math.inf                              # all of them listed
    if C > 1000:
        x[5, at[5][k:]] = -math.inf                         # and nothing else in the row
    got = losses.top_logits(x.cuda(), k, 2.0)
    some = losses.TopLogits(*(a[:6] for a in got))
    same_top(x[:6], k, 2.0, some)
    assert some.rest.isposinf().tolist() == [True] * 4 + [False] * 2 and some.rest.isnan().tolist() == [False] * 4 + [True, False]
    if rows == 6:                                           # the same as maps of three positions
        maps = losses.top_logits(x.view(2, 3, C).movedim(-1, 1).contiguous().cuda(), k, 2.0, dim=1)
        assert torch.equal(maps.indices.movedim(1, -1).reshape(6, k), some.indices)
        assert torch.equal(maps.rest.reshape(6).isposinf(), some.rest.isposinf()) and torch.equal(maps.rest.reshape(6).isnan(), some.rest.isnan())


@pytest.mark.gpu
def test_infinite_student_logits(hip_lib):
    """a logit of +inf has no softmax: its row's loss is NaN, whichever way the row is taken; other rows keep theirs"""
    from msf_wsi_amd import losses

    z = logits_of(4, 300, torch.float32, 1)
    v, i, r = to.top_logits(logits_of(4, 300, torch.float32, 2), 4, 1.0)
    z[1, int(i[1, 2])], z[2, (set(range(300)) - set(i[2].tolist())).pop()] = math.inf, math.inf
    for dim in (-1, 1):
        zl, vl, il = (a.t()[None].contiguous().cuda() if dim == 1 else a.cuda() for a in (z, v.float(), i.int()))
        zl.requires_grad_()
        row = losses.TopLogitDistillLoss(1.0, "none", dim=dim)(zl, losses.TopLogits(vl, il, r.float().cuda().view((1, 4) if dim == 1 else (4,))))
        grad, = torch.autograd.grad(row, zl, torch.ones_like(row))
        grad = grad[0].t() if dim == 1 else grad
        assert row.reshape(-1).isnan().tolist() == [False, True, True, False]
        assert grad.isnan().all(1).tolist() == [False, True, True, False] and bool(torch.isfinite(grad[[0, 3]]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
@pytest.mark.parametrize("kind", ["equal", "ascending", "descending", "far apart", "random"])
@pytest.mark.parametrize("C,k", [(70001, 1), (131072, 8), (70001, 40)])
def test_long_sums_of_one_lane(hip_lib, dt, kind, C, k):
    """maps give a lane all classes of a position: an addition at a time would lose n / 2 steps where the terms are alike.  The sums
    are taken 32 terms at a time and added with compensation, so 32 roundings (and 2) stand in the place of the n / 16 above."""
    from msf_wsi_amd import losses

    dt = FP[dt]
    if kind == "equal":                                     # behind two that are a little larger
        one = torch.zeros(C)
        one[0], one[1] = 0.3, 0.2
    elif kind == "ascending":
        one = torch.arange(C) / C
    elif kind == "descending":
        one = -torch.arange(C) / C
    elif kind == "far apart":                               # the reference of the sum moves again and again
        one = torch.arange(C) / C * 300 - 200
    else:
        one = torch.randn(C, generator=torch.Generator().manual_seed(C))
    x = torch.stack([one, one.roll(C // 2), one + 0.25, one.roll(77)]).to(dt)
    E = (3 * float((x.double().amax(1) - x.double().amin(1)).max()) + 34 + 64) * U
    maps = x.view(2, 2, C).movedim(-1, 1).contiguous().cuda()
    got = losses.top_logits(maps, k, dim=1)
    v, i = torch.sort(x.double(), dim=1, descending=True, stable=True)   # the definition, without a loop over 131072 classes
    i, r = i[:, :k], torch.logsumexp(v[:, k:], 1)
    assert torch.equal(got.indices.movedim(1, -1).reshape(4, k).cpu().long(), i)
    assert bool(((got.rest.reshape(4).cpu().double() - r).abs() <= E + 2 * U * r.abs()).all())
    teacher = losses.TopLogits(torch.zeros(2, k, 2, device="cuda"), torch.arange(k, dtype=torch.int32, device="cuda").view(1, k, 1).repeat(2, 1, 2))
    z = maps.requires_grad_()
    row = losses.TopLogitDistillLoss(1.0, "none", dim=1)(z, teacher)
    grad, = torch.autograd.grad(row, z, torch.ones_like(row))
    want, wgrad, _ = to.distill(x, torch.zeros(4, k), torch.arange(k).repeat(4, 1), None, None, 1.0)
    # the k entries' terms are added one by one, each addition off by U of a sum of at most the loss itself (here up to 302, U of which
    # times 40 is 7e-4, while E is 6e-5), each term by two roundings
    assert bool(((row.detach().reshape(4).cpu().double() - want).abs() <= E + (k + 2) * U * want.abs()).all())
    size = torch.softmax(x.double(), 1)
    size[:, :k] += 1.0 / k
    # An exponential below 2^-126 is 0 in the kernels and its factor T (q_r - p_r) here at most 1, so an element may be off by up to
    # 2^-126 (300 apart, the smallest q are e^-300: all elements past the tolerance without this term held less than 2^-126)
    tiny = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}[dt]
    err = (grad.movedim(1, -1).reshape(4, C).cpu().double() - wgrad).abs()
    assert bool((err <= 2 * E * size + torch.finfo(dt).eps / 2 * wgrad.abs() * (1 + 1e-5) + tiny).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", list(FP))
@pytest.mark.parametrize("small", [-68.5, -62.0, -60.5])
def test_rest_far_below_the_list(hip_lib, dt, small):
    """one class small enough that the thousands below it, each just too small for the list's scale, make a part of its size: a
    lane's 64 terms and the sums' tree are all that may be lost"""
    from msf_wsi_amd import losses

    C = 8192 if dt == "fp32" else 16384
    x = torch.full((3, C), -87.5)
    x[:, [5, 777, 2100, 4000]] = 0.0
    for r, at in enumerate((0, 3001, C - 1)):
        x[r, at] = small
    x = x.to(FP[dt])
    got = losses.top_logits(x.cuda(), 4)
    _, i, r = to.top_logits(x, 4, 1.0)
    assert torch.equal(got.indices.cpu().long(), i)
    assert bool(((got.rest.cpu().double() - r).abs() <= (3 * 87.5 + 128 + 64) * U + 2 * U * r.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["rows", "maps"])
@pytest.mark.parametrize("k", [2, 9, 40])
def test_gradient_keeps_the_last_bits(hip_lib, layout, k):
    """equal logits: every exponential is 1 and every sum exact, so what is left are the two reciprocals (2 U each), q_r's two products,
    the one with its share and the one with the gradient that arrives: 8 U of an unlisted class; of a listed one 4 U of q and of p"""
    from msf_wsi_amd import losses

    for C in (1000, 5003, 20011, 40003, 60000, 65535, 100003):
        z = torch.full((2, C), -0.75)
        i = (torch.arange(k) * 7).int().repeat(2, 1)
        zl, il = (a.t()[None].contiguous().cuda() if layout == "maps" else a.cuda() for a in (z, i))
        zl.requires_grad_()
        row = losses.TopLogitDistillLoss(1.0, "none", dim=1 if layout == "maps" else -1)(zl, losses.TopLogits(torch.zeros_like(il, dtype=torch.float32), il))
        grad, = torch.autograd.grad(row, zl, torch.ones_like(row))
        grad = (grad[0].t() if layout == "maps" else grad).double().cpu()
        listed = torch.zeros(C, dtype=torch.bool)
        listed[i[0].long()] = True
        assert float((grad[:, ~listed] - 1 / C).abs().max()) <= 8 * U / C, C
        assert float((grad[:, listed] - (1 / C - 1 / k)).abs().max()) <= 4 * U * (1 / C + 1 / k), C


@pytest.mark.gpu
def test_more_rows_than_a_launch_takes(hip_lib):
    """2^26 rows of a wave each are all the threads of one launch: selection, loss and gradient of a few more, either side of that row"""
    from msf_wsi_amd import losses

    rows, C, k = 2 ** 26 + 77, 20, 17
    pick = [0, 1, 2 ** 24 - 1, 2 ** 24, 2 ** 26 - 1, 2 ** 26, 2 ** 26 + 1, rows - 1]
    small = logits_of(len(pick), C, torch.bfloat16, 9)
    z = torch.zeros(rows, C, dtype=torch.bfloat16, device="cuda")
    z[pick] = small.cuda()
    teacher = losses.top_logits(z, k, 2.0)
    some = losses.TopLogits(*(a[pick] for a in teacher))
    same_top(small, k, 2.0, some)
    assert teacher.indices[3].tolist() == list(range(k)) and teacher.indices[rows - 2].tolist() == list(range(k))
    z[pick] = z[pick].flip(1)
    z.requires_grad_()
    weight = torch.zeros(rows, device="cuda")
    weight[pick] = 1.0
    row = losses.TopLogitDistillLoss(2.0, "none")(z, teacher)
    grad, = torch.autograd.grad(row, z, weight)
    check(small.flip(1), some.values, some.indices, some.rest, None, 2.0, row.detach()[pick], grad[pick], torch.bfloat16)
    assert float(grad[3].abs().max()) == 0.0 and float(grad[rows - 2].abs().max()) == 0.0


def test_too_many_classes_are_refused(hip_lib):
    """class counts that an int cannot step past (or hold at all) come back as errors before anything is launched"""
    import ctypes

    from msf_wsi_amd import kernels as kn

    for C in (2 ** 30 + 1, 2 ** 31 - 1, 2 ** 32 + 5):
        for shape in ((1, C), (2, C, 3)):
            with pytest.raises(ValueError):
                kn._logit_layout(torch.empty(shape, dtype=torch.bfloat16, device="meta"), "z")
    need, at = ctypes.c_long(), 4096                        # an address that nothing reads
    for C in (2 ** 30 + 1, 2 ** 31 - 1):
        assert hip_lib.msfwsi_top_logits_workspace(1, 1, C, 1, 2, ctypes.byref(need)) == -1
        assert hip_lib.msfwsi_top_logits(1, at, C, 1, C, 1, 2, 1.0, at, at, at, at, None) == -1
        assert hip_lib.msfwsi_distill_fwd(1, at, C, 1, C, 1, 2, at, at, None, None, 1.0, 1, at, None, at, at, at, None) == -1
        assert hip_lib.msfwsi_distill_bwd(1, at, C, 1, C, 1, 2, at, at, None, 1.0, at, None, at, 0, at, None) == -1


@pytest.mark.gpu
def test_hooknet_maps(hip_lib):
    """the framework's segmentation model as teacher and student: its maps go into selection and loss as they are, the gradient back
    into its weights"""
    from test_hooknet_gpu import CLASSES, _build, _inputs

    from msf_wsi_amd import losses

    teacher, student = _build().cuda().eval(), _build().cuda().train()
    x1, x2, _, m2 = (t.cuda() for t in _inputs())
    k, T, mask = 3, 2.0, (m2 != 0)
    with torch.no_grad():
        tl = teacher(x1, x2)[1]
        top = losses.top_logits(tl, k, T, dim=1)
    z = student(x1, x2)[1]
    z.retain_grad()
    row = losses.TopLogitDistillLoss(T, "none", dim=1)(z, top, mask)
    assert row.shape == mask.shape and z.shape[1] == CLASSES + 1
    row.sum().backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for n, p in student.named_parameters() if n.startswith("target_branch"))
    pick = torch.randint(0, mask.numel(), (300,), generator=torch.Generator().manual_seed(1)).cuda()

    def rows_of(a):
        return a.detach().movedim(1, -1).reshape(mask.numel(), -1)[pick].cpu()

    some = losses.TopLogits(rows_of(top.values), rows_of(top.indices), top.rest.reshape(-1)[pick].cpu())
    same_top(rows_of(tl), k, T, some)
    check(rows_of(z).to(z.dtype), some.values, some.indices, some.rest, mask.reshape(-1)[pick].cpu(), T, row.detach().reshape(-1)[pick], rows_of(z.grad), z.dtype)
